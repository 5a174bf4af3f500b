// lf_packed.hip.h — sequences of different lengths, one behind the other in one tensor, for the attention kernels
// (-DLF_PACKED=1): row i of Q, K, V, O [rows, heads, D] belongs to sequence n where offsets[n] <= i < offsets[n + 1].
//
// The work items are the tiles of a list that lf_packed_plan (lf_packed_plan.hip) leaves on the GPU: the host knows the
// number of rows and of sequences, not the lengths, and launches a workgroup per head and entry that the list can have.  A kernel takes its
// tile's sequence for the whole problem: B = 1, Sq = Sk = its length, pointers at its first row.
//   Workgroup -> (entry, head): the heads of an entry are neighbours, so that with a multiple of 8 of them each XCD walks
// its own heads over the entries in their order, and the tiles of a (sequence, head) share its K / V (or Q / dO) in one L2.  A list is
// ordered by the tiles' work within groups of sequences; which list a launch takes: packed.group_size.
//   MFMA- and exponential-bound as the dense kernels are, with the longest chain of tiles on top where sequences are few.  Kernels, bf16 causal, head
// dim 128, 12 sequences up to 2048, 32/8 heads: 177 us (877 TFLOP/s); window 256 and softcap, fp16, 5 up to 4001: 94 us (2.6 TB/s of Q, K, V and O);
// forward, delta, dK and dV, dQ, 8 up to 2048, 32/32 heads 142 + 41 + 322 + 102 us (631 TFLOP/s); forward, delta, all gradients, 24 up to 1000, fp16, D 64,
// 16/4 heads 25 + 11 + 66 us (its longest key tile).
//   P, and dS in the backward, are 16-bit operands of the second products, as in the dense kernels: matrix instructions take both operands in the
// type of K, V, Q and dO, and dS kept in 32 bits would be twice the bytes that bound dQ.  Against 64 bits that is 1.25 ... 1.45 times the error of
// rounding the results alone, a little over 1.5 where rows of dS cancel.
#ifndef LF_PACKED_HIP_H
#define LF_PACKED_HIP_H

struct LfPackedTile {
  int row0;        // first row of the sequence
  int len;         // its rows; 0: no tile
  int tile;        // number of the tile in it; a tile has as many rows as the list is for
  int seq;         // number of the sequence; -1: rows of no sequence
};
typedef const LfPackedTile __attribute__((address_space(4))) lf_ctile;

// the tile of an entry, through scalar loads
__device__ __forceinline__ LfPackedTile lf_packed_tile(const LfPackedTile* tiles, int entry) {
  const lf_ctile* t = reinterpret_cast<const lf_ctile*>(reinterpret_cast<unsigned long long>(tiles)) + entry;
  LfPackedTile r;
  r.row0 = t->row0;
  r.len = t->len;
  r.tile = t->tile;
  r.seq = t->seq;
  return r;
}

// Rows of no sequence: zeros into rows first .. first + rows - 1 (those below `end`) of `heads` neighbouring heads.
template <int NT>
__device__ __forceinline__ void lf_packed_clear(lf_elem* x, long long sh, long long ss, int heads, int first, int rows, int end) {
  constexpr int kChunks = LF_HEAD_DIM / 8;
  rows = min(rows, end - first);
  for (int i = threadIdx.x; i < rows * heads * kChunks; i += NT) {
    const int c = i % kChunks, h = i / kChunks % heads, r = i / (kChunks * heads);
    *reinterpret_cast<lf_u32x4*>(x + (long long)(first + r) * ss + h * sh + 8 * c) = lf_u32x4{0u, 0u, 0u, 0u};
  }
}

struct LfPackedAttnParams : LfAttnParams {      // Sq = Sk = rows of the tensors, B = 1
  const LfPackedTile* tiles;
  // Optional, strides of O: O in 32 bits minus O as stored, rounded.  The backward takes delta = rowsum(dO * O) from dP, often of its size:
  // of O as stored alone, dQ and dK are off by 1.8 times what rounding the formula's gradients costs, of both by 1.45 times.  The 2 bytes
  // per element, written and read once, cost 572 -> 597 us (forward and backward) at 8 sequences up to 2048, 32/32 heads of 128.
  lf_elem* low;
  int clear;               // 1: rows of no sequence are set to zero, 0: they are left as they are
};

#endif  // LF_PACKED_HIP_H
