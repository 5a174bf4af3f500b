// lf_rotate.hip — norms of queries and keys for each head and the rotation by their positions in one pass over them, into new tensors
// (LF_ROT_STORE 0), or with the keys and the values going into their slots of page pools, of 16-bit rows (1) or held in 4 bits (2);
// and the gradients.
//
// A head's row x of D elements: n = x / sqrt(mean(x^2) + eps), z = n * w (without a norm z = x); then with (c, s) the table's row of the token's
// position, for each of R / 2 pairs, (y0, y1) = (z0 c - z1 s, z1 c + z0 s); the other D - R elements stay.  In 32 bits, rounded once.  The rotation's
// products are rounded before they are summed (no fused multiply-add), as the same formula in a tensor language rounds them: what a cache in
// 4 bits takes for a row does not depend on who rotated it.
//
// LF_ROT_SLOTS threads have a row, 16 elements each: 8 of either half of what is rotated, or of the rest, so that no value changes threads
// but in the norm's sum (row permutations of 16 lanes) and a load or store of several threads has whole lines.  A group of threads takes two heads of a token, whose row of the table it
// reads once: one, two and four at a time took 134 / 129 / 133 us forwards and backwards together, 75 / 75 / 79 into pages and 50 / 48 / 50 into 4 bits and back, at the sizes below and
// before rows were read past the caches.  Reading them so took 128 to 125, 74 to 76, which is slower, and 53 to 49 over seconds of nothing else; 129 to 118, 75 to 66 and 49 to 48 in loops of 20 passes over other rows.
//
// Bound by memory.  Seconds of nothing else: 8192 rows of 32 and 32 heads of 128 in bf16 with norms, forwards and backwards with the weights' gradients, 126 us (671 MB, 5.3 TB/s); 16384 rows of 32 and 8 heads
// into pages 76 (407 MB, 5.3).  A kernel among 300 passes: the former's 43 forwards (268 MB, 6.2 TB/s) and 69 backwards (403 MB, 5.8), the latter 65 (6.2), 8192 such rows into 4 bits 37 (177 MB, 4.8).
// One new token each for up to 64 requests: 3.5 to 4.5 us, a launch and two round trips to memory.
//
// In 4 bits: 32 neighbours of a row share a power of two, 2^e with the least e of which their largest size is below 7 * 2^e (what lies between
// 6 and 7 of them rounds to 6, an error no larger than that of the step from 4 to 6), and each has a sign, two bits of exponent and one of mantissa
// (0 0.5 1 1.5 2 3 4 6), rounded to the nearest, ties to the even code.  Rows go through LDS for that, so that a thread has 8
// neighbours and four threads a block.  Where the codes lie is said in lf_pool4.hip.h.
#ifndef LF_ROT_STORE
#define LF_ROT_STORE 0
#endif
#define LF_ROT_HEADS 2
#define LF_ROT_SLOTS (LF_HEAD_DIM / 16)    /* 1, 2, 4, 8, 16: D rounded up to a power of two */
#define LF_ROT_NT 256
#define LF_ROT_GROUPS (LF_ROT_NT / LF_ROT_SLOTS)

struct LfRotateParams {
  const lf_elem* q;            // [T, Hq, D], strides below
  const lf_elem* k;            // [T, Hkv, D]
  const lf_elem* v;
  lf_elem* q_out;              // [T, Hq, D]
  void* k_out;                 // [T, Hkv, D], or the pool
  void* v_out;
  unsigned char* k_scales;     // of pools in 4 bits
  unsigned char* v_scales;
  const float* table;          // [places, R]: cosines, sines
  const void* q_weight;        // [D] or none
  const void* k_weight;
  const int* positions;        // [T]; none: all rows live, no rotation
  const int* slots;            // [T]
  long long q_ss, q_sh, k_ss, k_sh, v_ss, v_sh;        // rows, heads
  long long kp_sb, kp_ss, kp_sh, vp_sb, vp_ss, vp_sh;  // pages, tokens of a page, heads of the pools (LF_ROT_STORE 2: bytes of a page's codes, of its scales, unused)
  long long table_stride, last;                        // last: slots of a pool
  int T, Hq, Hkv, D, R, places;
  int q_chunks, k_chunks;      // groups of LF_ROT_HEADS heads
  int q_blocks, k_blocks;      // workgroups of the queries, of the keys; the others have values
  int shift;                   // log2 of the tokens per page
  int pairs, norm, wide;       // neighbours are partners; with norms; weights in 32 bits
  float eps;
};

struct LfRotateBwdParams {
  const lf_elem* q;            // as above (none without norms)
  const lf_elem* k;
  const lf_elem* dq_out;       // gradients of the results
  const lf_elem* dk_out;
  lf_elem* dq;                 // [T, Hq, D]
  lf_elem* dk;
  const float* table;
  const void* q_weight;
  const void* k_weight;
  void* dq_weight;             // [D], of the weights' type
  void* dk_weight;
  float* parts;                // [q_blocks + k_blocks, D], without weights none
  const int* positions;
  long long q_ss, q_sh, k_ss, k_sh, dqo_ss, dqo_sh, dko_ss, dko_sh;
  long long table_stride;
  int T, Hq, Hkv, D, R, places;
  int q_chunks, k_chunks, q_blocks, k_blocks;
  int pairs, norm, wide;
  float eps;
};

// sum over the threads of a row
__device__ __forceinline__ float lf_rot_sum(float x) {
  if (LF_ROT_SLOTS > 1) x += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0xb1, 0xf, 0xf, false));    // quad_perm [1,0,3,2]
  if (LF_ROT_SLOTS > 2) x += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x4e, 0xf, 0xf, false));    // quad_perm [2,3,0,1]
  if (LF_ROT_SLOTS > 4) x += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x141, 0xf, 0xf, false));   // row_half_mirror
  if (LF_ROT_SLOTS > 8) x += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x140, 0xf, 0xf, false));   // row_mirror
  return x;
}

// 1 / sqrt(x).  The instruction takes numbers below the least normal one for zeros: those are brought up by 2^24 first (without an eps elements of 2^-64 have such means).
__device__ __forceinline__ float lf_rot_root(float x) {
  const bool small = x < 0x1p-126f;
  return __builtin_amdgcn_rsqf(small ? x * 0x1p24f : x) * (small ? 0x1p12f : 1.0f);
}

// What a thread has of a row: 8 elements from `a` and 8 from `b`, of either half of the part that is rotated (`turns`) or of the rest, so that a load of several threads has whole lines.
struct LfRotPlace {
  int a, b;
  bool turns;
};
__device__ __forceinline__ LfRotPlace lf_rot_place(int slot, int R, int D) {
  const bool turns = 16 * slot < R;
  const int a = turns ? 8 * slot : R + 8 * (slot - R / 16);
  return {a, a + (turns ? R : D - R) / 2, turns};
}
__device__ __forceinline__ void lf_rot_load(const lf_elem* row, const LfRotPlace& at, lf_elem8 (&raw)[2]) {
  // (read once here)
  raw[0] = __builtin_nontemporal_load(reinterpret_cast<const lf_elem8*>(row + at.a));
  raw[1] = __builtin_nontemporal_load(reinterpret_cast<const lf_elem8*>(row + at.b));
}
__device__ __forceinline__ void lf_rot_floats(const lf_elem8 (&raw)[2], float (&x)[16]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] = lf_to_float(raw[i / 8][i % 8]);
}
__device__ __forceinline__ void lf_rot_store(lf_elem* row, const LfRotPlace& at, const float (&x)[16]) {
  lf_elem8 y[2];
#pragma unroll
  for (int i = 0; i < 16; ++i) y[i / 8][i % 8] = lf_from_float(x[i]);
  *reinterpret_cast<lf_elem8*>(row + at.a) = y[0];
  *reinterpret_cast<lf_elem8*>(row + at.b) = y[1];
}
__device__ __forceinline__ void lf_rot_weights(const void* w, int wide, const LfRotPlace& at, float (&x)[16]) {
  if (!w) {
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = 1.0f;
  } else if (wide) {
    const float* f = reinterpret_cast<const float*>(w);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const lf_f32x4 y = *reinterpret_cast<const lf_f32x4*>(f + (i < 2 ? at.a + 4 * i : at.b + 4 * (i - 2)));
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 * i + e] = y[e];
    }
  } else {
    const lf_elem* f = reinterpret_cast<const lf_elem*>(w);
    const lf_elem8 raw[2] = {*reinterpret_cast<const lf_elem8*>(f + at.a), *reinterpret_cast<const lf_elem8*>(f + at.b)};
    lf_rot_floats(raw, x);
  }
}
// cosines and sines of a thread's 8 pairs, which are one behind the other, or with neighbours as partners four of either half
__device__ __forceinline__ void lf_rot_angles(const float* row, int R, int pairs, int slot, float (&c)[8], float (&s)[8]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float* at = row + (pairs ? 4 * slot + i * (R / 4) : 8 * slot + 4 * i);
    const lf_f32x4 x = *reinterpret_cast<const lf_f32x4*>(at), y = *reinterpret_cast<const lf_f32x4*>(at + R / 2);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      c[4 * i + e] = x[e];
      s[4 * i + e] = y[e];
    }
  }
}
// (x0, x1) -> (x0 c - x1 s, x1 c + x0 s) for the thread's pairs, which lie 8 or 1 apart
template <int kApart>
__device__ __forceinline__ void lf_rot_turn(float (&x)[16], const float (&c)[8], const float (&s)[8]) {
#pragma clang fp contract(off)
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int j = kApart == 8 ? i : 2 * i;
    const float x0 = x[j], x1 = x[j + kApart];
    x[j] = x0 * c[i] - x1 * s[i];
    x[j + kApart] = x1 * c[i] + x0 * s[i];
  }
}

extern "C" __global__ void __launch_bounds__(LF_ROT_NT) lf_rotate(const LfRotateParams p) {
  const int tid = threadIdx.x, slot_of_row = tid % LF_ROT_SLOTS;
  int block = blockIdx.x;
  const int which = block < p.q_blocks ? 0 : block < p.q_blocks + p.k_blocks ? 1 : 2;      // queries, keys, values
  block -= which == 0 ? 0 : which == 1 ? p.q_blocks : p.q_blocks + p.k_blocks;
  const int H = which ? p.Hkv : p.Hq, chunks = which ? p.k_chunks : p.q_chunks, R = which == 2 ? 0 : p.R;
  const unsigned item = (unsigned)block * LF_ROT_GROUPS + tid / LF_ROT_SLOTS;
  const unsigned t = item / (unsigned)chunks;
  const int h0 = (int)(item - t * chunks) * LF_ROT_HEADS;
  const bool in = t < (unsigned)p.T && 16 * slot_of_row < p.D;
  const int position = t < (unsigned)p.T && p.positions ? p.positions[t] : 0;
  const bool live = in && position >= 0 && position < p.places;
  int slot = -1;
  if (LF_ROT_STORE && which && t < (unsigned)p.T && position >= 0 && position < p.places) {
    slot = p.slots[t];
    slot = slot < p.last ? slot : -1;
  }
  const LfRotPlace at = lf_rot_place(slot_of_row, R, p.D);
  const lf_elem* x0 = which == 0 ? p.q + (long long)t * p.q_ss : which == 1 ? p.k + (long long)t * p.k_ss : p.v + (long long)t * p.v_ss;
  const long long x_sh = which == 0 ? p.q_sh : which == 1 ? p.k_sh : p.v_sh;
  const bool wanted = live && (!LF_ROT_STORE || which == 0 || slot >= 0);
  lf_elem8 raw[LF_ROT_HEADS][2];
#pragma unroll
  for (int u = 0; u < LF_ROT_HEADS; ++u) {
    raw[u][0] = raw[u][1] = lf_elem8{};
    if (wanted && h0 + u < H) lf_rot_load(x0 + (h0 + u) * x_sh, at, raw[u]);
  }
  float c[8], s[8], w[16];
  if (wanted && at.turns) lf_rot_angles(p.table + (long long)position * p.table_stride, R, p.pairs, slot_of_row, c, s);
  const bool norm = p.norm && which != 2;
  if (norm && in) lf_rot_weights(which ? p.k_weight : p.q_weight, p.wide, at, w);
#if LF_ROT_STORE == 2
  __shared__ __attribute__((aligned(16))) lf_elem rows[LF_ROT_GROUPS][LF_HEAD_DIM + 8];
#endif
#pragma unroll
  for (int u = 0; u < LF_ROT_HEADS; ++u) {
    float x[16];
    lf_rot_floats(raw[u], x);
    if (norm) {
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < 16; ++i) sum += x[i] * x[i];
      const float r = lf_rot_root(lf_rot_sum(sum) / (float)p.D + p.eps);
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = x[i] * r * w[i];
    }
    if (wanted && at.turns) {
      if (p.pairs)
        lf_rot_turn<1>(x, c, s);
      else
        lf_rot_turn<8>(x, c, s);
    }
    const int h = h0 + u;
    if (which == 0 || !LF_ROT_STORE) {
      if (!wanted) {       // a row of no token
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = 0.0f;
      }
      if (in && h < H) lf_rot_store((which ? reinterpret_cast<lf_elem*>(p.k_out) : p.q_out) + ((long long)t * H + h) * p.D, at, x);
    } else {
#if LF_ROT_STORE == 1
      const long long page = slot >> p.shift, place = slot & ((1 << p.shift) - 1);
      lf_elem* pool = reinterpret_cast<lf_elem*>(which == 1 ? p.k_out : p.v_out);
      const long long sb = which == 1 ? p.kp_sb : p.vp_sb, ss = which == 1 ? p.kp_ss : p.vp_ss, sh = which == 1 ? p.kp_sh : p.vp_sh;
      if (wanted && h < H) lf_rot_store(pool + page * sb + place * ss + h * sh, at, x);
#elif LF_ROT_STORE == 2
      lf_wave_exchange();
      lf_rot_store(rows[tid / LF_ROT_SLOTS], at, x);
      lf_wave_exchange();
      // 2 LF_ROT_SLOTS threads a row, 8 neighbours each
      const int lane = tid & 63;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int row = half * (32 / LF_ROT_SLOTS) + lane / (2 * LF_ROT_SLOTS), r8 = lane % (2 * LF_ROT_SLOTS);
        const int its_slot = __shfl(slot, row * LF_ROT_SLOTS, 64), its_head = __shfl(h, row * LF_ROT_SLOTS, 64);
        const lf_elem8 y = *reinterpret_cast<const lf_elem8*>(&rows[(tid & ~63) / LF_ROT_SLOTS + row][8 * r8]);
        unsigned scale;
        const unsigned codes = lf_pool4_codes(y, scale);
        if (its_slot >= 0 && its_head < H)
          lf_pool4_put(which == 2, reinterpret_cast<unsigned char*>(which == 1 ? p.k_out : p.v_out), which == 1 ? p.k_scales : p.v_scales,
                       which == 1 ? p.kp_sb : p.vp_sb, which == 1 ? p.kp_ss : p.vp_ss, its_slot, p.shift, its_head, r8, codes, scale);
      }
#endif
    }
  }
}

#if LF_ROT_STORE == 0
// Gradients.  With g the gradient of y: dz = its rotation back, (g0 c + g1 s, g1 c - g0 s), dw = sum of dz n over rows, and with h = dz w
// dx = (h - n mean(h n)) / sqrt(mean(x^2) + eps).  Each workgroup sums dw over its share of the rows in registers, then over its threads, and leaves
// a part; lf_rotate_dw adds the parts, in an order that depends on the sizes alone.
extern "C" __global__ void __launch_bounds__(LF_ROT_NT) lf_rotate_bwd(const LfRotateBwdParams p) {
  const int tid = threadIdx.x, slot_of_row = tid % LF_ROT_SLOTS;
  const int which = (int)blockIdx.x < p.q_blocks ? 0 : 1;
  const int block = blockIdx.x - (which ? p.q_blocks : 0), blocks = which ? p.k_blocks : p.q_blocks;
  const int H = which ? p.Hkv : p.Hq, chunks = which ? p.k_chunks : p.q_chunks;
  const LfRotPlace at = lf_rot_place(slot_of_row, p.R, p.D);
  const lf_elem* x0 = which ? p.k : p.q;
  const lf_elem* g0 = which ? p.dk_out : p.dq_out;
  lf_elem* out = which ? p.dk : p.dq;
  const long long x_ss = which ? p.k_ss : p.q_ss, x_sh = which ? p.k_sh : p.q_sh, g_ss = which ? p.dko_ss : p.dqo_ss, g_sh = which ? p.dko_sh : p.dqo_sh;
  const bool inside = 16 * slot_of_row < p.D;
  float w[16], dw[16];
  if (p.norm && inside) lf_rot_weights(which ? p.k_weight : p.q_weight, p.wide, at, w);
#pragma unroll
  for (int i = 0; i < 16; ++i) dw[i] = 0.0f;
  const long long items = (long long)p.T * chunks;
  // (all threads of a workgroup make as many steps, as the norm's sums go over them)
  for (long long first = (long long)block * LF_ROT_GROUPS; first < items; first += (long long)blocks * LF_ROT_GROUPS) {
    const unsigned item = (unsigned)(first + tid / LF_ROT_SLOTS);
    const unsigned t = item / (unsigned)chunks;
    const int h0 = (int)(item - t * chunks) * LF_ROT_HEADS;
    const bool in = inside && t < (unsigned)p.T;
    const int position = in ? p.positions[t] : -1;
    const bool live = position >= 0 && position < p.places;
    lf_elem8 gr[LF_ROT_HEADS][2], xr[LF_ROT_HEADS][2];
#pragma unroll
    for (int u = 0; u < LF_ROT_HEADS; ++u) {
      gr[u][0] = gr[u][1] = xr[u][0] = xr[u][1] = lf_elem8{};
      if (live && h0 + u < H) {
        lf_rot_load(g0 + (long long)t * g_ss + (h0 + u) * g_sh, at, gr[u]);
        if (p.norm) lf_rot_load(x0 + (long long)t * x_ss + (h0 + u) * x_sh, at, xr[u]);
      }
    }
    float c[8], s[8];
    if (live && at.turns) lf_rot_angles(p.table + (long long)position * p.table_stride, p.R, p.pairs, slot_of_row, c, s);
#pragma unroll
    for (int u = 0; u < LF_ROT_HEADS; ++u) {
      float g[16];
      lf_rot_floats(gr[u], g);
      if (live && at.turns) {
        float back[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) back[i] = -s[i];
        if (p.pairs)
          lf_rot_turn<1>(g, c, back);
        else
          lf_rot_turn<8>(g, c, back);
      }
      if (p.norm) {
        float x[16], sum = 0.0f, dot = 0.0f;
        lf_rot_floats(xr[u], x);
#pragma unroll
        for (int i = 0; i < 16; ++i) sum += x[i] * x[i];
        // (where there is no row, or no such head, eps may be 0 and the root infinite: the zeros there stay zeros)
        const float y = lf_rot_sum(sum) / (float)p.D + p.eps, r = live && h0 + u < H ? lf_rot_root(y) : 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          x[i] *= r;
          dw[i] += g[i] * x[i];
          g[i] = inside ? g[i] * w[i] : 0.0f;
          dot += g[i] * x[i];
        }
        dot = lf_rot_sum(dot) / (float)p.D;
#pragma unroll
        for (int i = 0; i < 16; ++i) g[i] = (g[i] - x[i] * dot) * r;
      }
      if (!live) {
#pragma unroll
        for (int i = 0; i < 16; ++i) g[i] = 0.0f;
      }
      if (in && h0 + u < H) lf_rot_store(out + ((long long)t * H + h0 + u) * p.D, at, g);
    }
  }
  if (!p.parts) return;
  // over the groups of threads: a wave's by exchanges, then the four waves' through LDS
  __shared__ float sums[LF_ROT_NT / 64][LF_HEAD_DIM];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
#pragma unroll
    for (int d = LF_ROT_SLOTS; d < 64; d <<= 1) dw[i] += __shfl_xor(dw[i], d, 64);
  }
  if ((tid & 63) < LF_ROT_SLOTS && inside) {
#pragma unroll
    for (int i = 0; i < 16; ++i) sums[tid / 64][(i < 8 ? at.a : at.b) + i % 8] = dw[i];
  }
  __syncthreads();
  for (int d = tid; d < p.D; d += LF_ROT_NT) {
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < LF_ROT_NT / 64; ++i) sum += sums[i][d];
    p.parts[(long long)blockIdx.x * p.D + d] = sum;
  }
}

// dw of the parts: a workgroup has 16 columns of the queries' weight (blockIdx.y 0) or the keys', 4 to a thread, 64 threads to a column, which take every 64th
// part, eight loads under way at a time.  Bound by its chain of round trips: 2048 parts of 128 columns 24 us one part at a time.
extern "C" __global__ void __launch_bounds__(LF_ROT_NT) lf_rotate_dw(const LfRotateBwdParams p) {
  constexpr int kSplit = LF_ROT_NT / 4, kLook = 8;
  const int d = 16 * blockIdx.x + 4 * (threadIdx.x % 4), part = threadIdx.x / 4;
  const int first = blockIdx.y ? p.q_blocks : 0, count = blockIdx.y ? p.k_blocks : p.q_blocks;
  void* out = blockIdx.y ? p.dk_weight : p.dq_weight;
  if (!out) return;
  lf_f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int i = part; i < count; i += kLook * kSplit) {
    lf_f32x4 x[kLook];
#pragma unroll
    for (int u = 0; u < kLook; ++u) x[u] = *reinterpret_cast<const lf_f32x4*>(p.parts + (long long)(first + min(i + u * kSplit, count - 1)) * p.D + d);
#pragma unroll
    for (int u = 0; u < kLook; ++u)
      if (i + u * kSplit < count) sum += x[u];
  }
  __shared__ lf_f32x4 sums[kSplit][4];
  sums[part][threadIdx.x % 4] = sum;
  __syncthreads();
#pragma unroll
  for (int n = kSplit / 2; n >= 1; n /= 2) {
    if (part < n) sums[part][threadIdx.x % 4] += sums[part + n][threadIdx.x % 4];
    __syncthreads();
  }
  if (part) return;
  sum = sums[0][threadIdx.x];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (p.wide)
      reinterpret_cast<float*>(out)[d + e] = sum[e];
    else
      reinterpret_cast<lf_elem*>(out)[d + e] = lf_from_float(sum[e]);
  }
}
#endif
