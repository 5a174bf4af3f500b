// lf_packed_positions.hip — the place of each packed row in its sequence, -1 for rows of none.
// A thread has a row and looks for the last sequence that begins at it or before, by halves; the offsets are in L1 after the first steps.  Bound by that chain: log2(sequences) loads
// from L2, once per batch for all layers.
struct LfPackedPositionsParams {
  const int* offsets;          // [N + 1]
  int* positions;              // [T]
  int N, T;
};

extern "C" __global__ void __launch_bounds__(256) lf_packed_positions(const LfPackedPositionsParams p) {
  const unsigned row = blockIdx.x * 256 + threadIdx.x;
  if (row >= (unsigned)p.T) return;
  int lo = 0, hi = p.N + 1;    // offsets before lo are at most row, those from hi on more
  while (lo < hi) {
    const int mid = lo + (hi - lo) / 2;
    if (p.offsets[mid] <= (int)row)
      lo = mid + 1;
    else
      hi = mid;
  }
  // (of several that begin there the last is the one that is not empty)
  p.positions[row] = lo == 0 || lo > p.N ? -1 : (int)row - max(p.offsets[lo - 1], 0);
}
