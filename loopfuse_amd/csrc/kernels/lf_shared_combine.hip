// lf_shared_combine.hip — joins the partial results of attention over a shared prefix and over the requests' own keys.
// A block = 256 threads = 1024 / D rows (a row: request, query head) of one request, a thread owns 4 consecutive d of one.  Parts of
// a row: the prefix's splits, then the request's pieces, four at a time: their loads go out together.  Bound by that chain of
// round trips.  A row without a part, i.e. without a key, gives zeros.
extern "C" __global__ void __launch_bounds__(256) lf_shared_combine(const LfSharedParams p) {
  constexpr int kTPR = LF_HEAD_DIM / 4, kRPB = 256 / kTPR;
  const int heads = p.Hkv * p.rows, per = (heads + kRPB - 1) / kRPB;
  const int b = blockIdx.x / per, head = (blockIdx.x % per) * kRPB + threadIdx.x / kTPR;
  const int d0 = 4 * (threadIdx.x % kTPR);
  int first, count;
  lf_shared_pieces_of(p, lf_shared_split(p), b, first, count);
  if (head >= heads || (p.Sk == 0 && count == 1)) return;       // (one piece and nothing else: written already)
  const int hkv = head / p.rows, qr = head % p.rows;
  const int splits = p.Sk ? p.nsplit : 0, parts = splits + count;
  const long long pre = (long long)hkv * p.nsplit * p.B * p.rows + (long long)b * p.rows + qr;
  float m = LF_NEG_INF, l = 0.0f;
  lf_f32x4 a = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int z0 = 0; z0 < parts; z0 += 4) {
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
    float mc = m;
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (z0 + u < parts) mc = fmaxf(mc, ml[u][0]);
    const float m_sub = (mc == LF_NEG_INF) ? 0.0f : mc;
    const float r = (m == LF_NEG_INF) ? 0.0f : lf_exp2(m - m_sub);
    l *= r;
    a *= r;
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (z0 + u < parts) {
        const float f = lf_exp2(ml[u][0] - m_sub);
        l += ml[u][1] * f;
        a += ac[u] * f;
      }
    m = mc;
  }
  const float inv = parts ? lf_inv_sum(l) : 0.0f;
  lf_elem4 w;
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = lf_from_float(a[e] * inv);
  *reinterpret_cast<lf_elem4*>(p.o + (long long)b * p.o_sb + (long long)hkv * p.o_sh + (long long)qr * p.o_ss + d0) = w;
}
