// lf_cached.hip — attention of the new tokens of requests of different lengths over their keys and values in page pools held in 4 bits
// (lf_pool4.hip.h), those of the new tokens among them.
//
// Request b has n = offsets[b + 1] - offsets[b] rows of q and lengths[b] keys; a row at position p sees the keys j <= p (and p - j < window), or all.
// A unit of work is a kv head's LF_CACHED_ROWS rows of a request over its keys, 32 at a time.  Lengths are on the GPU only: every wave sums what the units
// cost, each its pairs of tiles of 16 keys and something for its begin, and finds the share of its workgroup, the same for all, by itself.  So no workgroup
// waits for a longer one.  A unit that several workgroups have leaves, from each, an exponent offset, the sum of the exponentials and their sum with V per
// row, which lf_cached_combine joins; one that a workgroup has alone is written at once.  Where units are many each workgroup takes one.
//
// A wave takes 32 keys at a time for LF_CACHED_CB * 16 rows:
//   S^T = K Q^T   : lane (key c, g) has elements D / 4 * g ... of its key, which share a power of two: conversions of two codes at a time, exact in the rows' type, make first operands
//                   of the 16x16x32 products of them, eight elements a step; lane (q = c, g) has the same elements of Q.  (The products of 4- with 8-bit numbers that take powers of two
//                   along would save these conversions, q in two 8-bit parts, but what they sum is cut off 2^-12 below the largest product, where keys with a few large elements need it.)
//                   Lane (q = c, g) receives S^T[keys 4 g ... 4 g + 3][q].
//   softmax       : one exponent offset per row, which may lag the running maximum by 2^LF_CACHED_LAZY.
//   O^T += V^T P^T: a lane holds 4 keys' D / 16 neighbouring elements; two conversions and two byte permutations make the two lanes' worth of operand of two elements out of them, and the
//                   product number i has the elements D / 16 * row + i, so that a lane ends up with D / 4 neighbouring elements of O.
//
// Few rows: 16 of a kv head, or 32, a workgroup's four waves have a fourth of the pairs of tiles each and merge through LDS in the end; operands straight from memory, two pairs under way, no LDS
// and no barrier in the loop.  Bound by memory where keys are many: 64 requests of one token up to 8192 keys, 32/8 heads of 128, 53 us and 5 for the joining (291 MB, 5.0 TB/s both); 4 up to
// 100 000 47 and 5 (272 MB, 5.2); by one wave's chain where they are few: 2 up to 1000 10 us, 16 700 cycles of a wave: lengths and shares 2600, the first loads 2300, eight pairs 9800, the merge 1700; 48 requests of five new tokens in a
// window of 1024 with a cap, 16/4 heads of 64, 15 us, 25 400 cycles: 3800, 3800, 14 300, 3000.  Of either's cycles waves wait in 0.47 and issue in 0.43.
// By conversions, softmax and products in between: 64 up to 8192 with five new tokens each 74 us, 32 rows at a time (16: 99).
// Many rows (LF_CACHED_ROWWAVES): 128, each wave has 32 of them over all pairs.  Of a pair two waves convert a tile of keys each, two one of values, into LDS, where all four find the operands as the
// products take them: a fourth of the conversions, and fewer registers, so that three waves run on a SIMD.  Bound by the softmax and the products: 4 requests up to 6001 keys with up to 1000
// new tokens 230 us (213 GFLOP, 926 TFLOP/s; each wave with keys and values of its own 257), 2 of 8192 with 4096 805 us (1025; 897).
#ifndef LF_CACHED_CB
#define LF_CACHED_CB 1
#endif
#ifndef LF_CACHED_ROWWAVES
#define LF_CACHED_ROWWAVES 0
#endif
#define LF_CACHED_LAZY 8
#define LF_CACHED_ROWS (16 * LF_CACHED_CB * (LF_CACHED_ROWWAVES ? 4 : 1))     /* of a workgroup */
#define LF_CACHED_NV (LF_HEAD_DIM / 16)    /* products of O^T */
#define LF_CACHED_OSTRIDE (LF_HEAD_DIM + 4)


struct LfCachedParams {
  const lf_elem* q;            // [T, Hq, D], strides below
  lf_elem* o;
  const unsigned char* k;      // codes and scales of the pools
  const unsigned char* v;
  const unsigned char* k_scales;
  const unsigned char* v_scales;
  const void* table;           // [B, ...], rows table_stride apart
  const int* lengths;          // [B]
  const int* offsets;          // [B + 1]; none: a row each
  const int* positions;        // [T]; none: the last key's
  float* part_acc;             // [slots, LF_CACHED_ROWS, D]
  float* part_ml;              // [slots, LF_CACHED_ROWS, 2]
  long long q_ss, q_sh, o_ss, o_sh;
  long long page_bytes, table_stride;                  // of codes, for keys and values alike, 16 times those of scales; entries
  int T, B, Hkv, group;
  unsigned per_group;          // 2^32 / group, rounded up
  int room;                    // keys that a row of the table has room for
  int shift;                   // log2 of the tokens per page
  int window;
  int fixed;                   // what a unit costs besides its pairs of tiles, in pairs; below 0: each workgroup has a unit, whatever it costs
  int least;                   // least share of a workgroup
  int workgroups;
  int slots;                   // that there is room for, as many as the units and workgroups; offsets that descend would ask for more: those stay away
  int clear;                   // 1: zeros into rows of no request
  float scale, softcap;
};

// A request: its rows and its keys.
struct LfCachedRequest {
  int first, n;
  int start, end;              // the first key that any row can see, a multiple of 32; the last one's successor
  int chunks;                  // LF_CACHED_ROWS rows of a kv head each
  int pairs;                   // of tiles of 16 keys, 1 at least: a unit without a key has its zeros to write
};
__device__ __forceinline__ LfCachedRequest lf_cached_request(const LfCachedParams& p, int b) {
  LfCachedRequest r;
  const int at = min(b, p.B - 1);
  int end = p.lengths[at], lo = at, hi = at + 1;
  if (p.offsets) {
    lo = p.offsets[at];
    hi = p.offsets[at + 1];
  }
  r.first = min(max(lo, 0), p.T);
  r.n = b < p.B ? max(min(hi, p.T) - r.first, 0) : 0;
  r.end = min(max(end, 0), p.room);
  r.start = 0;
#if LF_MASK == 2
  const int from = p.positions && r.n > 0 ? max(p.positions[r.first], 0) : r.end - 1;
  r.start = min(max(from - p.window + 1, 0), max(r.end - 1, 0)) & ~31;
#endif
  r.chunks = (int)(((long long)r.n * p.group + LF_CACHED_ROWS - 1) / LF_CACHED_ROWS);
  r.pairs = max((r.end - r.start + 31) >> 5, 1);
  return r;
}

// The units (request, chunk, kv head), heads innermost, lie one behind the other on a line, each as long as `fixed` and its pairs (or all of length 1);
// workgroup i has the line from i * share on.  (The host sees to it that the line is shorter than 2^31.)
__device__ __forceinline__ int lf_cached_size(const LfCachedParams& p, const LfCachedRequest& r) { return p.fixed < 0 ? 1 : r.pairs + p.fixed; }
__device__ __forceinline__ int lf_cached_line(const LfCachedParams& p, const LfCachedRequest& mine) {
  int line = 0;
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    const LfCachedRequest r = b0 ? lf_cached_request(p, b0 + __lane_id()) : mine;
    line += __builtin_amdgcn_readlane(lf_wave_scan(r.chunks * p.Hkv * lf_cached_size(p, r)), 63);
  }
  return line;
}
__device__ __forceinline__ int lf_cached_share(const LfCachedParams& p, int line, int workgroups) { return max(p.least, (line + workgroups - 1) / workgroups); }

struct LfCachedPlace {
  int b;
  LfCachedRequest r;
  int before;                  // on the line, in front of the request's units
  int units;                   // of the requests in front of it
};
__device__ __forceinline__ void lf_cached_take(const LfCachedRequest& r, int lane, LfCachedPlace& u) {
  u.r.first = __builtin_amdgcn_readlane(r.first, lane);
  u.r.n = __builtin_amdgcn_readlane(r.n, lane);
  u.r.start = __builtin_amdgcn_readlane(r.start, lane);
  u.r.end = __builtin_amdgcn_readlane(r.end, lane);
  u.r.chunks = __builtin_amdgcn_readlane(r.chunks, lane);
  u.r.pairs = __builtin_amdgcn_readlane(r.pairs, lane);
}
// The request that has place `place` of the line, or where that is below 0 row `row`; false: none has.
__device__ __forceinline__ bool lf_cached_find(const LfCachedParams& p, const LfCachedRequest& mine, int place, int row, LfCachedPlace& u) {
#if LF_CACHED_ROWWAVES
  if (p.fixed < 0 && p.B <= 64) {
    // a unit each: those of the request with the most keys first, as what begins last should be short
    const int count = mine.chunks * p.Hkv, lane = __lane_id();
    int before = 0;
    for (int i = 0; i < p.B; ++i) {
      const int pairs = __builtin_amdgcn_readlane(mine.pairs, i), its = __builtin_amdgcn_readlane(count, i);
      if (pairs > mine.pairs || (pairs == mine.pairs && i < lane)) before += its;
    }
    const unsigned long long hit = __builtin_amdgcn_ballot_w64(place >= before && place < before + count);
    if (hit == 0ull) return false;
    lf_cached_take(mine, (int)__builtin_ctzll(hit), u);
    u.b = (int)__builtin_ctzll(hit);
    u.before = __builtin_amdgcn_readlane(before, u.b);
    u.units = 0;
    return true;
  }
#endif
  int before = 0, units = 0;
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    const LfCachedRequest r = b0 ? lf_cached_request(p, b0 + __lane_id()) : mine;
    const int count = r.chunks * p.Hkv, cost = count * lf_cached_size(p, r), upto = lf_wave_scan(cost), units_upto = lf_wave_scan(count);
    const unsigned long long hit = __builtin_amdgcn_ballot_w64(place >= 0 ? before + upto > place : r.n > 0 && row >= r.first && row < r.first + r.n);
    if (hit != 0ull) {
      const int l = (int)__builtin_ctzll(hit);
      u.b = b0 + l;
      lf_cached_take(r, l, u);
      u.before = before + __builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(cost, l);
      u.units = units + __builtin_amdgcn_readlane(units_upto, l) - __builtin_amdgcn_readlane(count, l);
      return true;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
    units += __builtin_amdgcn_readlane(units_upto, 63);
  }
  return false;
}

// Largest, or least, over the 16 lanes of a row, the same in all four rows of the wave.
template <bool kMost>
__device__ __forceinline__ int lf_cached_of_rows(int x) {
  auto take = [](int a, int b) { return kMost ? max(a, b) : min(a, b); };
  x = take(x, __builtin_amdgcn_update_dpp(x, x, 0xb1, 0xf, 0xf, false));       // quad_perm [1,0,3,2]
  x = take(x, __builtin_amdgcn_update_dpp(x, x, 0x4e, 0xf, 0xf, false));       // quad_perm [2,3,0,1]
  x = take(x, __builtin_amdgcn_update_dpp(x, x, 0x141, 0xf, 0xf, false));      // row_half_mirror
  x = take(x, __builtin_amdgcn_update_dpp(x, x, 0x140, 0xf, 0xf, false));      // row_mirror
  return __builtin_amdgcn_readfirstlane(x);
}

// 32 keys of a head as loaded
typedef unsigned lf_cached_codes __attribute__((ext_vector_type(LF_HEAD_DIM / 32)));
#if LF_CACHED_ROWWAVES
struct LfCachedStage {
  lf_cached_codes x;           // of this wave's tile: of a key D / 4 neighbours, or of four keys' values D / 16 neighbours each
  unsigned scales;
};
#else
struct LfCachedStage {
  lf_cached_codes k[2];        // of a key D / 4 neighbours
  lf_cached_codes v[2];        // of four keys D / 16 neighbours each
  unsigned ks[2], vs[2];
};
#endif

extern "C" __global__ void __launch_bounds__(256, LF_CACHED_ROWWAVES && LF_HEAD_DIM == 64 ? 4 : LF_CACHED_ROWWAVES || LF_CACHED_CB == 1 ? 3 : 2) lf_cached(const LfCachedParams p) {
  constexpr int D = LF_HEAD_DIM, CB = LF_CACHED_CB, NJ = D / 32;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, g = lane >> 4;
  const LfCachedRequest mine = lf_cached_request(p, lane);
  const int line = lf_cached_line(p, mine), share = lf_cached_share(p, line, p.workgroups);
  auto inverse = [](float l) { return l == 0.0f ? 0.0f : 1.0f / l; };      // a row without a key: zeros; NaN stays
#if LF_CACHED_ROWWAVES
  // 32 keys as operands of the products, twice
  __shared__ lf_elem8 kt[2][2][NJ][64];                    // [tile, step][lane]
  __shared__ lf_elem4 vt[2][LF_CACHED_NV][2][64];          // [product][tile][lane]
  __shared__ unsigned v_scales_of[2][2][64];               // where a value is NaN
  __shared__ int v_nan[2][2], chunk_end[4], chunk_begin[4];
#else
  __shared__ float red_o[4 * 16 * LF_CACHED_OSTRIDE];
  __shared__ float red_m[4][16], red_l[4][16];
#endif
  int place = min((long long)blockIdx.x * share, (long long)line);
  const int place_end = min((long long)place + share, (long long)line);
  while (place < place_end) {
  LfCachedPlace u;
  if (!lf_cached_find(p, mine, place, 0, u)) break;
  const int size = lf_cached_size(p, u.r), unit = (place - u.before) / size, from = place - u.before - unit * size, upto = min(size, from + place_end - place);
  // (under a causal mask the last rows have the most keys: first)
  const int chunk = u.r.chunks - 1 - unit / p.Hkv, h = unit % p.Hkv;
  const int slot = u.units + unit + (int)blockIdx.x;       // (either grows along the line)
  place += upto - from;
  if (upto <= p.fixed) continue;
  const int pair0 = p.fixed < 0 ? 0 : max(from - p.fixed, 0), pair1 = p.fixed < 0 ? u.r.pairs : upto - p.fixed;
  const int rows = u.r.n * p.group;      // of a kv head
  const int row0 = chunk * LF_CACHED_ROWS + (LF_CACHED_ROWWAVES ? wave * 16 * CB : 0);
  const bool whole = pair0 == 0 && pair1 == u.r.pairs;
  if (!whole && (unsigned)slot >= (unsigned)p.slots) break;

  // ---- loads: rows of this lane, one per column block, and their positions; then the first keys
  lf_elem8 qb[CB][NJ];
  int pos[CB];
#pragma unroll
  for (int cb = 0; cb < CB; ++cb) {
    // (rows behind the last repeat the chunk's first; their results are dropped)
    const int row = row0 + 16 * cb + c, at = row < rows ? row : min(row0, rows - 1);
    const int t_of = p.group == 1 ? at : (int)__umulhi((unsigned)at, p.per_group);
    const int t = u.r.first + t_of, head = h * p.group + at - t_of * p.group;
    pos[cb] = p.positions ? p.positions[t] : u.r.end - 1;
    const lf_elem* qrow = p.q + (long long)t * p.q_ss + head * p.q_sh + D / 4 * g;
#pragma unroll
    for (int j = 0; j < NJ; ++j) qb[cb][j] = *reinterpret_cast<const lf_elem8*>(qrow + 8 * j);
  }
  int begin = u.r.start + 32 * pair0, pairs = u.r.end > 0 ? pair1 - pair0 : 0;
  const int last_tile = max(u.r.end - 1, 0) & ~15;
  const int head_tiles = h << (p.shift - 4);
  const int in_page = (1 << p.shift) - 1;
#if LF_TABLE_I64
  const lf_cu64* ids = reinterpret_cast<const lf_cu64*>(reinterpret_cast<unsigned long long>(p.table)) + (long long)u.b * p.table_stride;
#else
  const lf_cint* ids = reinterpret_cast<const lf_cint*>(reinterpret_cast<unsigned long long>(p.table)) + (long long)u.b * p.table_stride;
#endif
  auto tile_of = [&](int pair, int which) { return min(begin + 32 * min(pair, pairs - 1) + 16 * which, last_tile); };
  const int k_at = c * (D / 2) + D / 8 * g, ks_at = (c * D + D / 4 * g) / 32, v_at = D / 8 * lane, vs_at = (g * (D / 32) + c / (512 / D)) * 4;
#if LF_CACHED_ROWWAVES
  // two waves have the keys' tiles, two the values'
  const int tile_w = wave & 1;
  const bool has_values = wave >= 2;
  const unsigned char* codes_of = has_values ? p.v : p.k;
  const unsigned char* scales_of = has_values ? p.v_scales : p.k_scales;
  const unsigned x_at = has_values ? v_at : k_at, scales_at = has_values ? vs_at : ks_at;
  auto issue = [&](LfCachedStage& s, int pair) {
    const int tile = tile_of(pair, tile_w);
    const long long codes = (int)ids[tile >> p.shift] * p.page_bytes + (head_tiles + ((tile & in_page) >> 4)) * (8 * D);
    s.x = *reinterpret_cast<const lf_cached_codes*>(codes_of + codes + x_at);
    if (has_values)
      s.scales = *reinterpret_cast<const unsigned*>(scales_of + (codes >> 4) + scales_at);
    else
      s.scales = scales_of[(codes >> 4) + scales_at];
  };
  // what was loaded into the operands' places
  auto convert = [&](LfCachedStage& s, int pair, int buf) {
    if (!has_values) {
      const float by = __builtin_bit_cast(float, s.scales << 23);
#pragma unroll
      for (int j = 0; j < NJ; ++j) kt[buf][tile_w][j][lane] = lf_pool4_values(s.x[j], by);
      return;
    }
    const int t0 = begin + 32 * pair + 16 * tile_w;
    if (t0 + 16 > u.r.end) {
      // what lies behind the last key may be anything: nothing, with weights of zero
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e >= u.r.end - t0 - 4 * g) s.scales &= ~(0xffu << (8 * e));
    }
    const bool nan = ((~s.scales - 0x01010101u) & s.scales & 0x80808080u) != 0u, any = __builtin_amdgcn_ballot_w64(nan) != 0ull;
    if (any) {
      v_scales_of[buf][tile_w][lane] = s.scales;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (((s.scales >> (8 * e)) & 0xffu) == 0xffu) s.scales &= ~(0xffu << (8 * e));
    }
    if (lane == 0) v_nan[buf][tile_w] = any;
    float by[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) by[e] = __builtin_bit_cast(float, e == 3 ? s.scales >> 1 : s.scales << (23 - 8 * e));       // (only a power's exponent is looked at)
#pragma unroll
    for (int m = 0; m < LF_CACHED_NV / 2; ++m) {
      lf_elem4 va[2];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const unsigned word = s.x[D == 128 ? e : e / 2];
        lf_pool4_two y;
        switch (D == 128 ? m : 2 * (e % 2) + m) {
          case 0: y = lf_pool4_pair<0>(word, by[e]); break;
          case 1: y = lf_pool4_pair<1>(word, by[e]); break;
          case 2: y = lf_pool4_pair<2>(word, by[e]); break;
          default: y = lf_pool4_pair<3>(word, by[e]);
        }
        va[0][e] = y[0];
        va[1][e] = y[1];
      }
      vt[buf][2 * m][tile_w][lane] = va[0];
      vt[buf][2 * m + 1][tile_w][lane] = va[1];
    }
  };
#else
  constexpr int kStep = 4;
  const int first = wave;
  // Codes that are not in a cache the next time anyhow pass the caches by: from 128 MB on, as the line counts them.  That is each request's keys once for each chunk of its rows, and `fixed` pairs more for every
  // unit: more than there are where requests are short or have several chunks.  us, kept / by: 4 requests up to 100 000 keys 58.4 / 52.1, 64 up to 8192 64.2 / 57.7, 16 of 8000 (139 MB) 35.7 / 33.3;
  // 8 of 8000 (70 MB) 20.7 / 21.6, 4 of 8192 with 4 new tokens (36 MB) 18.3 / 19.5.  By the line, but not by their codes, beyond it: 256 of 128 in wide tables (35 MB) 28.8 / 32.1,
  // 8 of 8000 with 10 new tokens (70 MB, two chunks) 36.2 / 39.9.
  constexpr int kStream = (128 << 20) / (34 * D);       // pairs of tiles
  struct Ids {
    int a, b;                  // (a pool has less than 2^31 pages)
  };
  auto fetch = [&](int pair) -> Ids { return {(int)ids[tile_of(pair, 0) >> p.shift], (int)ids[tile_of(pair, 1) >> p.shift]}; };
  const bool streams = p.fixed >= 0 && line >= kStream;
  auto issue = [&](LfCachedStage& s, int pair, const Ids& id) {
    long long codes[2];
#pragma unroll
    for (int w = 0; w < 2; ++w) codes[w] = (w ? id.b : id.a) * p.page_bytes + (head_tiles + ((tile_of(pair, w) & in_page) >> 4)) * (8 * D);
    if (streams) {
      asm volatile("; streams");       // (or the compiler makes one load of both)
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        s.k[w] = __builtin_nontemporal_load(reinterpret_cast<const lf_cached_codes*>(p.k + codes[w] + k_at));
        s.v[w] = __builtin_nontemporal_load(reinterpret_cast<const lf_cached_codes*>(p.v + codes[w] + v_at));
      }
      asm volatile("; streams");
    } else {
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        s.k[w] = *reinterpret_cast<const lf_cached_codes*>(p.k + codes[w] + k_at);
        s.v[w] = *reinterpret_cast<const lf_cached_codes*>(p.v + codes[w] + v_at);
      }
    }
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      s.ks[w] = p.k_scales[(codes[w] >> 4) + ks_at];
      s.vs[w] = *reinterpret_cast<const unsigned*>(p.v_scales + (codes[w] >> 4) + vs_at);
    }
  };
#endif
  // loads past the end repeat the last pair, so that there is no condition on them
#if LF_CACHED_ROWWAVES
  LfCachedStage s;
#else
  // (two stages take turns)
  LfCachedStage s0, s1;
  Ids i0, i1;
  auto issue_first = [&]() {
    if (first >= pairs) return;
    i0 = fetch(first);
    i1 = fetch(first + kStep);
    issue(s0, first, i0);
    issue(s1, first + kStep, i1);
    i0 = fetch(first + 2 * kStep);
    i1 = fetch(first + 3 * kStep);
  };
  issue_first();
#endif
  // bounds of the rows
  int lo[CB], hi[CB];
  int least_hi = 0x7fffffff, most_hi = 0, least_lo = 0x7fffffff, most_lo = 0;
#pragma unroll
  for (int cb = 0; cb < CB; ++cb) {
    hi[cb] = pos[cb] < 0 ? 0 : LF_MASK == 0 ? u.r.end : min(pos[cb], u.r.end - 1) + 1;
    lo[cb] = LF_MASK == 2 ? max(max(pos[cb], 0) - p.window + 1, 0) : 0;
    least_hi = min(least_hi, hi[cb]);
    most_hi = max(most_hi, hi[cb]);
    least_lo = min(least_lo, lo[cb]);
    most_lo = max(most_lo, lo[cb]);
  }
  least_hi = lf_cached_of_rows<false>(least_hi);
  if (LF_MASK == 2) most_lo = lf_cached_of_rows<true>(most_lo);
#if LF_CACHED_ROWWAVES
  // (what no row of the chunk sees is left out)
  const int wave_end = lf_cached_of_rows<true>(most_hi), wave_begin = LF_MASK == 2 ? lf_cached_of_rows<false>(least_lo) : 0;
  if (lane == 0) {
    chunk_end[wave] = wave_end;
    chunk_begin[wave] = wave_begin;
  }
  __syncthreads();
  {
    const int ends = min(begin + 32 * pairs, max(max(chunk_end[0], chunk_end[1]), max(chunk_end[2], chunk_end[3])));
    if (LF_MASK == 2) begin = max(begin, min(min(chunk_begin[0], chunk_begin[1]), min(chunk_begin[2], chunk_begin[3])) & ~31);
    pairs = ends > begin ? (ends - begin + 31) >> 5 : 0;
    pairs = __builtin_amdgcn_readfirstlane(pairs);
    begin = __builtin_amdgcn_readfirstlane(begin);
  }
  if (pairs > 0) issue(s, 0);
#endif

#if LF_SOFTCAP
  const float sc_in = p.scale / p.softcap;
  const float cexp = LF_LOG2E;
#else
  const float cexp = p.scale * LF_LOG2E;
#endif
  lf_f32x4 o[CB][LF_CACHED_NV];
  float mc[CB], l_part[CB], bad[CB];
#pragma unroll
  for (int cb = 0; cb < CB; ++cb) {
    mc[cb] = LF_NEG_INF;
    l_part[cb] = bad[cb] = 0.0f;
#pragma unroll
    for (int i = 0; i < LF_CACHED_NV; ++i) o[cb][i] = lf_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }

  // ---- 32 keys
#if LF_CACHED_ROWWAVES
  auto consume = [&](int buf, int pair) {
#else
  auto consume = [&](LfCachedStage& s, int pair) {
#endif
    const int t0 = begin + 32 * pair;
    const bool partly = t0 < most_lo || t0 + 32 > least_hi;      // some row does not see all of them
#if LF_CACHED_ROWWAVES
    const int nan0 = v_nan[buf][0], nan1 = v_nan[buf][1];
#else
    if (t0 + 32 > u.r.end) {
      // what lies behind the last key may be anything: nothing, with weights of zero
#pragma unroll
      for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (t0 + 16 * w + 4 * g + e >= u.r.end) s.vs[w] &= ~(0xffu << (8 * e));
    }
    if (partly) {
      // values that are NaN must not meet a row that does not see them, whose weight of zero would make NaN of them: they count as zeros, and what a lane
      // has of the rows that do see them, neighbours of one block, becomes NaN in the end
      auto none = [](unsigned x) { return (~x - 0x01010101u) & x & 0x80808080u; };       // is a byte of it 255?
      if (__builtin_amdgcn_ballot_w64((none(s.vs[0]) | none(s.vs[1])) != 0u) != 0ull) {
        const int from = D / 4 * g / 32 * (512 / D);       // a lane that reads the scales of this one's block
#pragma unroll 1
        for (int i = 0; i < 8; ++i) {
          const unsigned byte = 0xffu << (8 * (i & 3));
          const bool mine = ((i < 4 ? s.vs[0] : s.vs[1]) & byte) == byte;
          const unsigned long long all = __builtin_amdgcn_ballot_w64(mine);
          if (mine) (i < 4 ? s.vs[0] : s.vs[1]) &= ~byte;
#pragma unroll
          for (int at = 0; at < 4; ++at) {
            const int t = t0 + 16 * (i >> 2) + 4 * at + (i & 3);
            const bool is = ((all >> (16 * at + from)) & 1) != 0;
#pragma unroll
            for (int cb = 0; cb < CB; ++cb)
              if (is && t >= lo[cb] && t < hi[cb]) bad[cb] = __builtin_nanf("");
          }
        }
      }
    }
#endif
    lf_f32x4 r[CB][2];
#pragma unroll
    for (int w = 0; w < 2; ++w) {
#if !LF_CACHED_ROWWAVES
      const float by = __builtin_bit_cast(float, s.ks[w] << 23);
#endif
#pragma unroll
      for (int cb = 0; cb < CB; ++cb) r[cb][w] = lf_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
#if LF_CACHED_ROWWAVES
        const lf_elem8 a = kt[buf][w][j][lane];
#else
        const lf_elem8 a = lf_pool4_values(s.k[w][j], by);
#endif
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) r[cb][w] = lf_mfma16(a, qb[cb][j], r[cb][w]);
      }
    }
    float top[CB];
    bool grows = false;
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) {
#if LF_SOFTCAP
#pragma unroll
      for (int i = 0; i < 8; ++i) r[cb][i / 4][i % 4] = p.softcap * lf_tanh(r[cb][i / 4][i % 4] * sc_in);
#endif
      if (partly) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int j = 16 * (i / 4) + i % 4;       // from t0 + 4 g on
          if (j >= hi[cb] - t0 - 4 * g || (LF_MASK == 2 && j < lo[cb] - t0 - 4 * g)) r[cb][i / 4][i % 4] = LF_NEG_INF;
        }
      }
      float mx = LF_NEG_INF;
#pragma unroll
      for (int i = 0; i < 8; ++i) mx = fmaxf(mx, r[cb][i / 4][i % 4]);
      top[cb] = mx * cexp;
      grows = grows || top[cb] > mc[cb] + (float)LF_CACHED_LAZY;
    }
    if (__builtin_amdgcn_ballot_w64(grows) != 0ull) {
#pragma unroll
      for (int cb = 0; cb < CB; ++cb) {
        float mq = fmaxf(top[cb], __shfl_xor(top[cb], 16, 64));
        mq = fmaxf(mq, __shfl_xor(mq, 32, 64));
        const float m_new = fmaxf(mc[cb], mq);
        const float f = (m_new == LF_NEG_INF) ? 1.0f : lf_exp2(mc[cb] - m_new);
        mc[cb] = m_new;
        l_part[cb] *= f;
#pragma unroll
        for (int i = 0; i < LF_CACHED_NV; ++i) o[cb][i] *= f;
      }
    }
    lf_elem8 pb[CB];
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) {
      const float m_sub = (mc[cb] == LF_NEG_INF) ? 0.0f : mc[cb];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float e = lf_exp2(__builtin_fmaf(r[cb][i / 4][i % 4], cexp, -m_sub));
        l_part[cb] += e;
        // (the second product's operand, so of the rows' type; two such parts of it would be twice the products.  Relative 2-norm against 64 bits 2.1e-3 to 2.3e-3 in bf16 and 2.8e-4 in fp16, where the
        // result's own rounding is 1.7e-3 and 2.1e-4)
        pb[cb][i] = lf_from_float(e);
      }
    }
#if LF_CACHED_ROWWAVES
#pragma unroll
    for (int i = 0; i < LF_CACHED_NV; ++i) {
      const lf_elem4 a = vt[buf][i][0][lane], b = vt[buf][i][1][lane];
      const lf_elem8 va = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
      for (int cb = 0; cb < CB; ++cb) o[cb][i] = lf_mfma16(va, pb[cb], o[cb][i]);
    }
    if ((__builtin_amdgcn_readfirstlane(nan0 | nan1)) != 0) {
      // values that are NaN must not meet a row that does not see them, whose weight of zero would make NaN of them: they count as zeros, and what a lane
      // has of the rows that do see them, neighbours of one block, becomes NaN in the end
      const int from = D / 4 * g / 32 * (512 / D);       // a lane that reads the scales of this one's block
#pragma unroll 1
      for (int i = 0; i < 32; ++i) {
        const int w = i >> 4, at = i & 15, t = t0 + i;
        const bool is = v_nan[buf][w] != 0 && ((v_scales_of[buf][w][16 * (at >> 2) + from] >> (8 * (at & 3))) & 0xffu) == 0xffu;
#pragma unroll
        for (int cb = 0; cb < CB; ++cb)
          if (is && t >= lo[cb] && t < hi[cb]) bad[cb] = __builtin_nanf("");
      }
    }
#else
    // V^T: lane (row c, g) has keys 4 g ... of either tile, elements D / 16 * c + 2 m and + 1 of byte m of each key
    float by[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) by[e] = __builtin_bit_cast(float, e % 4 == 3 ? s.vs[e / 4] >> 1 : s.vs[e / 4] << (23 - 8 * (e % 4)));       // (only a power's exponent is looked at)
#pragma unroll
    for (int m = 0; m < LF_CACHED_NV / 2; ++m) {
      lf_elem8 va[2];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const unsigned word = s.v[e / 4][D == 128 ? e % 4 : e % 4 / 2];
        lf_pool4_two y;
        switch (D == 128 ? m : 2 * (e % 2) + m) {
          case 0: y = lf_pool4_pair<0>(word, by[e]); break;
          case 1: y = lf_pool4_pair<1>(word, by[e]); break;
          case 2: y = lf_pool4_pair<2>(word, by[e]); break;
          default: y = lf_pool4_pair<3>(word, by[e]);
        }
        va[0][e] = y[0];
        va[1][e] = y[1];
      }
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) o[cb][2 * m + n] = lf_mfma16(va[n], pb[cb], o[cb][2 * m + n]);
    }
#endif
  };

#if LF_CACHED_ROWWAVES
  // ---- the workgroup's pairs: while a pair's products are formed the next one's operands go into the other places, and the one's after that are under way
  auto meet = [&]() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
  auto step = [&](int buf, int pr) {
    convert(s, pr + 1, buf ^ 1);
    issue(s, pr + 2);
    const int t0 = begin + 32 * pr;
    if (t0 < wave_end && (LF_MASK != 2 || t0 + 32 > wave_begin)) consume(buf, pr);
    meet();
  };
  if (pairs > 0) {
    convert(s, 0, 0);
    issue(s, 1);
    meet();
    for (int pr = 0; pr < pairs; pr += 2) {
      step(0, pr);
      if (pr + 1 >= pairs) break;
      step(1, pr + 1);
    }
  } else {
    __syncthreads();       // (the chunk's bounds are read)
  }
#else
  // ---- this wave's pairs
  for (int pr = first; pr < pairs; pr += 2 * kStep) {
    consume(s0, pr);
    issue(s0, pr + 2 * kStep, i0);
    i0 = fetch(pr + 4 * kStep);
    if (pr + kStep >= pairs) break;
    consume(s1, pr + kStep);
    issue(s1, pr + 3 * kStep, i1);
    i1 = fetch(pr + 5 * kStep);
  }
#endif
#pragma unroll
  for (int cb = 0; cb < CB; ++cb)
#pragma unroll
    for (int i = 0; i < LF_CACHED_NV; ++i) o[cb][i] += bad[cb];

  // ---- results: lane (q = c, g) has elements D / 4 * g ... of its row, 4 groups of D / 16
  float l_wave[CB];
#pragma unroll
  for (int cb = 0; cb < CB; ++cb) {
    l_wave[cb] = l_part[cb] + __shfl_xor(l_part[cb], 16, 64);
    l_wave[cb] += __shfl_xor(l_wave[cb], 32, 64);
  }
  const long long slot0 = (long long)slot * LF_CACHED_ROWS;
  auto out_row = [&](int row) {
    const unsigned t = p.group == 1 ? row : __umulhi(row, p.per_group);
    return p.o + (long long)(u.r.first + (int)t) * p.o_ss + (h * p.group + row - (int)t * p.group) * p.o_sh;
  };
#if LF_CACHED_ROWWAVES
#pragma unroll
  for (int cb = 0; cb < CB; ++cb) {
    const int row = row0 + 16 * cb + c;
    if (row >= rows) continue;
    if (whole) {
      lf_elem* to = out_row(row) + D / 4 * g;
      const float inv = inverse(l_wave[cb]);
#pragma unroll
      for (int n = 0; n < D / 32; ++n) {
        lf_elem8 y;
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = lf_from_float(o[cb][(8 * n + i) % LF_CACHED_NV][(8 * n + i) / LF_CACHED_NV] * inv);
        *reinterpret_cast<lf_elem8*>(to + 8 * n) = y;
      }
    } else {
      const long long at = slot0 + (row - chunk * LF_CACHED_ROWS);
#pragma unroll
      for (int n = 0; n < D / 16; ++n) {
        lf_f32x4 y;
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = o[cb][(4 * n + i) % LF_CACHED_NV][(4 * n + i) / LF_CACHED_NV];
        *reinterpret_cast<lf_f32x4*>(&p.part_acc[at * D + D / 4 * g + 4 * n]) = y;
      }
      if (g == 0) {
        p.part_ml[at * 2] = mc[cb];
        p.part_ml[at * 2 + 1] = l_wave[cb];
      }
    }
  }
#else
#pragma unroll
  for (int cb = 0; cb < CB; ++cb) {
    __syncthreads();       // (a block of rows, or a unit, before)
    if (g == 0) {
      red_m[wave][c] = mc[cb];
      red_l[wave][c] = l_wave[cb];
    }
    __syncthreads();
    {
      const float m_all = fmaxf(fmaxf(red_m[0][c], red_m[1][c]), fmaxf(red_m[2][c], red_m[3][c]));
      const float f = lf_exp2(mc[cb] - (m_all == LF_NEG_INF ? 0.0f : m_all));
#pragma unroll
      for (int n = 0; n < D / 16; ++n) {
        lf_f32x4 y;
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = o[cb][(4 * n + i) % LF_CACHED_NV][(4 * n + i) / LF_CACHED_NV] * f;
        *reinterpret_cast<lf_f32x4*>(&red_o[(wave * 16 + c) * LF_CACHED_OSTRIDE + D / 4 * g + 4 * n]) = y;
      }
    }
    __syncthreads();
    // thread -> (row, 8 elements)
    for (int at = tid; at < 16 * D / 8; at += 256) {
      const int r = at / (D / 8), d0 = at % (D / 8) * 8, row = row0 + 16 * cb + r;
      if (row >= rows) continue;
      const float m_all = fmaxf(fmaxf(red_m[0][r], red_m[1][r]), fmaxf(red_m[2][r], red_m[3][r])), m_sub = m_all == LF_NEG_INF ? 0.0f : m_all;
      float l = 0.0f, sum[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[i] = 0.0f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        l += red_l[w][r] * lf_exp2(red_m[w][r] - m_sub);
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[i] += red_o[(w * 16 + r) * LF_CACHED_OSTRIDE + d0 + i];
      }
      if (whole) {
        const float inv = inverse(l);
        lf_elem8 y;
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = lf_from_float(sum[i] * inv);
        *reinterpret_cast<lf_elem8*>(out_row(row) + d0) = y;
      } else {
        const long long to = slot0 + 16 * cb + r;
#pragma unroll
        for (int i = 0; i < 2; ++i)
          *reinterpret_cast<lf_f32x4*>(&p.part_acc[to * D + d0 + 4 * i]) = lf_f32x4{sum[4 * i], sum[4 * i + 1], sum[4 * i + 2], sum[4 * i + 3]};
        if (d0 == 0) {
          p.part_ml[to * 2] = m_all;
          p.part_ml[to * 2 + 1] = l;
        }
      }
    }
  }
#endif
  }
  if (p.clear && p.offsets) {
    // rows of no request, dealt to all workgroups
    const int lo = min(max(p.offsets[0], 0), p.T), hi = max(min(max(p.offsets[p.B], 0), p.T), lo);
    const int pieces = p.Hkv * p.group * (D / 8);
    const long long all = (long long)(lo + p.T - hi) * pieces;
    for (long long i = (long long)blockIdx.x * 256 + tid; i < all; i += (long long)gridDim.x * 256) {
      const long long row = i / pieces;
      const int at = (int)(i - row * pieces), head = at / (D / 8);
      *reinterpret_cast<lf_u32x4*>(p.o + (row < lo ? row : row - lo + hi) * p.o_ss + head * p.o_sh + 8 * (at - head * (D / 8))) = lf_u32x4{0u, 0u, 0u, 0u};
    }
  }
}

// Joins the parts of rows whose unit several workgroups have.  D / 4 threads have a row, 4 elements each; a block of 256 has 1024 / D heads of one token,
// or, in grids of a block per (token, head), one row whose parts its groups of threads share and merge through LDS.
extern "C" __global__ void __launch_bounds__(256) lf_cached_combine(const LfCachedParams p) {
  constexpr int kTPR = LF_HEAD_DIM / 4, kRPB = 256 / kTPR;
  const int Hq = p.Hkv * p.group;
  const bool row_per_block = (long long)gridDim.x == (long long)p.T * Hq;
  const int group = threadIdx.x / kTPR, per = row_per_block ? Hq : (Hq + kRPB - 1) / kRPB;
  const int t = blockIdx.x / per, head = row_per_block ? blockIdx.x - t * per : (blockIdx.x - t * per) * kRPB + group;
  const int d0 = 4 * (threadIdx.x % kTPR);
  const LfCachedRequest mine = lf_cached_request(p, __lane_id());
  const int share = lf_cached_share(p, lf_cached_line(p, mine), p.workgroups);
  LfCachedPlace u;
  if (!lf_cached_find(p, mine, -1, t, u) || head >= Hq) return;
  const int h = head / p.group, row = (t - u.r.first) * p.group + head - h * p.group, chunk = row / LF_CACHED_ROWS;
  const int unit = (u.r.chunks - 1 - chunk) * p.Hkv + h, size = u.r.pairs + p.fixed, place = u.before + unit * size;
  // the workgroups that have a pair of the unit
  const int first = (place + p.fixed) / share, parts = (place + size - 1) / share - first + 1;
  if (parts <= 1) return;        // (written already)
  const unsigned begin = u.units + unit + first;
  if (begin >= (unsigned)p.slots || (unsigned)parts > (unsigned)p.slots - begin) return;
  const long long slot0 = (long long)begin * LF_CACHED_ROWS + row - chunk * LF_CACHED_ROWS;
  float m = LF_NEG_INF, l = 0.0f;
  lf_f32x4 a = {0.0f, 0.0f, 0.0f, 0.0f};
  auto join = [&](float m2, float l2, const lf_f32x4& a2) {
    if (l2 == 0.0f) return;
    const float mj = fmaxf(m, m2), ms = mj == LF_NEG_INF ? 0.0f : mj, r = lf_exp2(m - ms), f = lf_exp2(m2 - ms);
    l = l * r + l2 * f;
    a = a * r + a2 * f;
    m = mj;
  };
  for (int z0 = row_per_block ? 4 * group : 0; z0 < parts; z0 += row_per_block ? 4 * kRPB : 4) {
    lf_f32x2 ml[4];
    lf_f32x4 ac[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const long long slot = slot0 + (long long)min(z0 + i, parts - 1) * LF_CACHED_ROWS;
      ml[i] = *reinterpret_cast<const lf_f32x2*>(&p.part_ml[slot * 2]);
      ac[i] = *reinterpret_cast<const lf_f32x4*>(&p.part_acc[slot * LF_HEAD_DIM + d0]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (z0 + i < parts) join(ml[i][0], ml[i][1], ac[i]);
  }
  if (row_per_block) {
    __shared__ lf_f32x4 acc[kRPB][kTPR];
    __shared__ lf_f32x2 ml[kRPB];
    acc[group][d0 / 4] = a;
    if (d0 == 0) ml[group] = lf_f32x2{m, l};
    __syncthreads();
    if (group) return;
#pragma unroll
    for (int i = 1; i < kRPB; ++i) join(ml[i][0], ml[i][1], acc[i][d0 / 4]);
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  lf_elem4 y;
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = lf_from_float(a[i] * inv);
  *reinterpret_cast<lf_elem4*>(p.o + (long long)t * p.o_ss + head * p.o_sh + d0) = y;
}
