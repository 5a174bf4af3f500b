// lf_packed_plan.hip — the tile lists of a packed batch (lf_packed.hip.h) from its offsets.
//
// Four lists, for tiles of 32, 64, 128 and 256 rows.  Sequences come in the order of their lengths, the longest first
// (equal ones in their own order), the tiles of one together: workgroups are dispatched in this order, so that the long ones
// do not come last.  Behind them the rows of no sequence (in front of the first offset, behind the last one), then empty entries.
//   Place of a sequence's first tile = tiles of the sequences in front of it in that order: every thread forms that sum for its own
// sequence by looking at all N lengths, 256 at a time through LDS.  N^2 / 256 steps per block, of which there are N / 256 per list:
// no sort, no scan across blocks, one launch.
// Whatever the offsets hold, tiles lie inside the T rows and places inside the list: offsets are clamped to 0 .. T, and what
// overlapping sequences have too many of is left out.

struct LfPackedPlanParams {
  const int* offsets;          // [N + 1]
  LfPackedTile* tiles;         // the four lists, one behind the other
  int N, T;
  int cap[4];                  // entries of each
};

#define LF_PLAN_NT 256
extern "C" __global__ void __launch_bounds__(LF_PLAN_NT) lf_packed_plan(const LfPackedPlanParams p) {
  __shared__ int s_len[LF_PLAN_NT], s_tiles[LF_PLAN_NT];
  const int list = blockIdx.y, shift = 5 + list, up = (1 << shift) - 1;
  LfPackedTile* out = p.tiles;
  for (int i = 0; i < list; ++i) out += p.cap[i];
  const int cap = p.cap[list];
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
  // places in front of this item, tiles of all sequences
  long long first = 0;
  for (int base = 0; base < p.N; base += LF_PLAN_NT) {
    const int j = base + threadIdx.x;
    const int l = j < p.N ? max(at(j + 1) - at(j), 0) : 0;
    __syncthreads();
    s_len[threadIdx.x] = l;
    s_tiles[threadIdx.x] = (l + up) >> shift;
    __syncthreads();
    const int count = min(p.N - base, LF_PLAN_NT);
    for (int i = 0; i < count; ++i) {
      const int other = s_len[i];
      if (n >= p.N || other > len || (other == len && base + i < n)) first += s_tiles[i];
    }
  }
  if (n == p.N + 1) first += (p.T - at(p.N) + up) >> shift;
  const int tiles = (len + up) >> shift;
  const bool last = n == p.N + 1;
  // entries are written by whole waves, one item after the other
  const int lane = threadIdx.x & 63;
  for (int i = 0; i < 64; ++i) {
    const int item = __builtin_amdgcn_readlane(n, i);
    if (item > p.N + 1) break;
    const int f = __builtin_amdgcn_readlane((int)min(first, (long long)cap), i), c = __builtin_amdgcn_readlane(tiles, i);
    const int r = __builtin_amdgcn_readlane(row0, i), l = __builtin_amdgcn_readlane(len, i);
    for (int t = lane; t < c && f + t < cap; t += 64) out[f + t] = LfPackedTile{r, l, t, item < p.N ? item : -1};
    if (__builtin_amdgcn_readlane((int)last, i))
      for (int t = f + c + lane; t < cap; t += 64) out[t] = LfPackedTile{0, 0, 0, -1};
  }
}
