// lf_packed_plan.hip — the tile lists of a packed batch (lf_packed.hip.h) from its offsets, in two launches.
//
// Lists for tiles of 32, 64, 128 and 256 rows (dispatch order = list order).  Sequences are sorted by length, the longest first (equal ones
// in their own order), and taken in groups of neighbours of 1, 2, 4 or 8, a list for each: in a group the tiles come by their work under
// a causal mask, the longest first, where tile t of a sequence of n tiles counts n - t (the kernels number them so).  One group for all would
// balance best and share the least in L2, groups of one the other way round; who launches knows how many heads an XCD has at a time.  Behind
// the sequences come the rows of no sequence (in front of the first offset, behind the last one), then empty entries.
//   lf_packed_sort: the rank of a sequence and the tiles in front of it, each a sum over all sequences that every thread forms for its own one:
// N^2 / 256 steps per block, N / 256 blocks, no scan across them.
//   lf_packed_plan: a wave per group; the place of tile t of the group's member g, with c = n_g - t, is the tiles in front of the group +
// sum_j max(0, n_j - c) (longer ones) + g (of those that are as long, the members before it).
// Whatever the offsets hold, tiles lie inside the T rows and places inside the list: offsets are clamped to 0 .. T, and what
// overlapping sequences have too many of is left out.
//   Bound by its chain of round trips (offsets, sums, stores): 2.3 + 3.8 us for 3 sequences, 3.6 + 5.1 for 12 up to 2048 rows, 4.6 + 5.2 for 24 up to
// 1000, once per batch for all layers, forward and backward.

#define LF_PLAN_LISTS 4        /* tile heights */
#define LF_PLAN_GROUPS 4       /* 1, 2, 4, 8 */
struct LfPackedPlanParams {
  const int* offsets;          // [N + 1]
  LfPackedTile* tiles;         // lists [height][group size][cap[height]]
  int* sorted;                 // [3 + LF_PLAN_LISTS][N + 2], of a rank: first row, rows, number of the sequence, tiles of each height in front of it
  int N, T;
  int cap[LF_PLAN_LISTS];
};

#define LF_PLAN_NT 256
extern "C" __global__ void __launch_bounds__(LF_PLAN_NT) lf_packed_sort(const LfPackedPlanParams p) {
  __shared__ int s_len[LF_PLAN_NT];
  const int M = p.N + 2;
  auto at = [&](int n) { return min(max(p.offsets[n], 0), p.T); };
  // item n < N: a sequence; N: the rows behind the last; N + 1: those in front of the first
  const int n = blockIdx.x * LF_PLAN_NT + threadIdx.x;
  int row0 = 0, len = 0;
  if (n < p.N) {
    row0 = at(n);
    len = max(at(n + 1) - row0, 0);
  } else if (n == p.N) {
    row0 = at(p.N);
    len = p.T - row0;
  } else if (n == p.N + 1) {
    len = at(0);
  }
  int rank = 0;
  long long first[LF_PLAN_LISTS] = {0, 0, 0, 0};
  for (int base = 0; base < p.N; base += LF_PLAN_NT) {
    const int j = base + threadIdx.x;
    const int l = j < p.N ? max(at(j + 1) - at(j), 0) : 0;
    __syncthreads();
    s_len[threadIdx.x] = l;
    __syncthreads();
    const int count = min(p.N - base, LF_PLAN_NT);
    for (int i = 0; i < count; ++i) {
      const int other = s_len[i];
      if (n >= p.N || other > len || (other == len && base + i < n)) {
        ++rank;
#pragma unroll
        for (int k = 0; k < LF_PLAN_LISTS; ++k) first[k] += (other + (32 << k) - 1) >> (5 + k);
      }
    }
  }
  if (n == p.N + 1) {
    ++rank;
#pragma unroll
    for (int k = 0; k < LF_PLAN_LISTS; ++k) first[k] += (p.T - at(p.N) + (32 << k) - 1) >> (5 + k);
  }
  if (n >= M) return;
  p.sorted[rank] = row0;
  p.sorted[M + rank] = len;
  p.sorted[2 * M + rank] = n;
#pragma unroll
  for (int k = 0; k < LF_PLAN_LISTS; ++k) p.sorted[(3 + k) * M + rank] = (int)min(first[k], (long long)p.cap[k]);
}

// grid: (blocks of 4 groups, heights x group sizes)
extern "C" __global__ void __launch_bounds__(LF_PLAN_NT) lf_packed_plan(const LfPackedPlanParams p) {
  const int height = blockIdx.y / LF_PLAN_GROUPS, size = 1 << (blockIdx.y % LF_PLAN_GROUPS);
  const int M = p.N + 2, shift = 5 + height, up = (1 << shift) - 1, cap = p.cap[height];
  LfPackedTile* out = p.tiles;
  for (int i = 0; i < height; ++i) out += (long long)LF_PLAN_GROUPS * p.cap[i];
  out += (long long)(blockIdx.y % LF_PLAN_GROUPS) * cap;
  const int lane = threadIdx.x & 63, wave = blockIdx.x * (LF_PLAN_NT / 64) + (threadIdx.x >> 6);
  const int groups = (p.N + size - 1) / size;
  const int* first = p.sorted + (3 + height) * M;
  if (wave < groups) {
    const int r0 = wave * size, members = min(size, p.N - r0), at = first[r0];
    int n[1 << (LF_PLAN_GROUPS - 1)];
#pragma unroll
    for (int j = 0; j < 1 << (LF_PLAN_GROUPS - 1); ++j) n[j] = j < members ? (p.sorted[M + r0 + j] + up) >> shift : 0;
#pragma unroll
    for (int g = 0; g < 1 << (LF_PLAN_GROUPS - 1); ++g) {
      if (g >= members) break;
      const int row0 = p.sorted[r0 + g], len = p.sorted[M + r0 + g], seq = p.sorted[2 * M + r0 + g];
      for (int t = lane; t < n[g]; t += 64) {
        const int c = n[g] - t;
        long long place = (long long)at + g;
#pragma unroll
        for (int j = 0; j < 1 << (LF_PLAN_GROUPS - 1); ++j) place += max(n[j] - c, 0);
        if (place < cap) out[place] = LfPackedTile{row0, len, t, seq};
      }
    }
  } else if (wave < groups + 2) {       // rows of no sequence; the second of the two also leaves the empty entries
    const int r = p.N + wave - groups, row0 = p.sorted[r], len = p.sorted[M + r], at = first[r], n = (len + up) >> shift;
    for (int t = lane; t < n; t += 64)
      if ((long long)at + t < cap) out[at + t] = LfPackedTile{row0, len, t, -1};
    if (wave == groups + 1)
      for (long long t = (long long)at + n + lane; t < cap; t += 64) out[t] = LfPackedTile{0, 0, 0, -1};
  }
}
