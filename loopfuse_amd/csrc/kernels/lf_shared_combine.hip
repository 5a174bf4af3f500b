// lf_shared_combine.hip — joins the partial results of attention over a shared prefix and over the requests' own keys.
// A thread owns 4 consecutive d of a row (a row: request, query head), so that D / 4 threads read a part's row whole.  A block of 256 has
// 1024 / D rows of one request, or, in grids of a block per row, one row whose parts its groups of threads share and merge through LDS.
// Parts of a row: the prefix's splits, then the request's pieces, four at a time per group: their loads go out together.  Bound by that
// chain of round trips where rows are few, by the partials' bytes where they are many: 32 heads of 128, 2 requests 3.2 us, 64 4.6, 128 6.2.
// A row without a part, i.e. without a key, gives zeros.
extern "C" __global__ void __launch_bounds__(256) lf_shared_combine(const LfSharedParams p) {
  constexpr int kTPR = LF_HEAD_DIM / 4, kRPB = 256 / kTPR;
  const int heads = p.Hkv * p.rows;
  const bool row_per_block = (int)gridDim.x == p.B * heads;      // (with kRPB == heads == 1 row either way)
  const int group = threadIdx.x / kTPR, per = row_per_block ? heads : (heads + kRPB - 1) / kRPB;
  const int b = blockIdx.x / per, head = row_per_block ? blockIdx.x % per : blockIdx.x % per * kRPB + group;
  const int d0 = 4 * (threadIdx.x % kTPR);
  const int mine = lf_shared_length(p, __lane_id());
  int first, count;
  lf_shared_pieces_of(p, mine, lf_shared_split(p, mine), b, first, count);
  if (head >= heads || (p.Sk == 0 && count == 1)) return;       // (one piece and nothing else: written already)
  const int hkv = head / p.rows, qr = head % p.rows;
  const int splits = p.Sk ? p.nsplit : 0, parts = splits + count;
  const long long pre = (long long)hkv * p.nsplit * p.B * p.rows + (long long)b * p.rows + qr;
  float m = LF_NEG_INF, l = 0.0f;
  lf_f32x4 a = {0.0f, 0.0f, 0.0f, 0.0f};
  auto join = [&](float m2, float l2, const lf_f32x4& a2) {
    if (m2 == LF_NEG_INF) return;
    const float mc = fmaxf(m, m2), r = (m == LF_NEG_INF) ? 0.0f : lf_exp2(m - mc), f = lf_exp2(m2 - mc);
    l = l * r + l2 * f;
    a = a * r + a2 * f;
    m = mc;
  };
  for (int z0 = row_per_block ? 4 * group : 0; z0 < parts; z0 += row_per_block ? 4 * kRPB : 4) {
    lf_f32x2 ml[4];
    lf_f32x4 ac[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int z = min(z0 + u, parts - 1);
      const bool own = z >= splits;
      const long long slot = own ? ((long long)(first + z - splits) * p.Hkv + hkv) * p.rows + qr : pre + (long long)z * p.B * p.rows;
      ml[u] = *reinterpret_cast<const lf_f32x2*>((own ? p.part_ml : p.pre_ml) + slot * 2);
      ac[u] = *reinterpret_cast<const lf_f32x4*>((own ? p.part_acc : p.pre_acc) + slot * LF_HEAD_DIM + d0);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (z0 + u < parts) join(ml[u][0], ml[u][1], ac[u]);
  }
  if (row_per_block) {
    __shared__ lf_f32x4 acc[kRPB][kTPR];
    __shared__ lf_f32x2 ml[kRPB];
    acc[group][d0 / 4] = a;
    if (d0 == 0) ml[group] = lf_f32x2{m, l};
    __syncthreads();
    if (group) return;
#pragma unroll
    for (int g = 1; g < kRPB; ++g) join(ml[g][0], ml[g][1], acc[g][d0 / 4]);
  }
  const float inv = parts ? lf_inv_sum(l) : 0.0f;
  lf_elem4 w;
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = lf_from_float(a[e] * inv);
  *reinterpret_cast<lf_elem4*>(p.o + (long long)b * p.o_sb + (long long)hkv * p.o_sh + (long long)qr * p.o_ss + d0) = w;
}
