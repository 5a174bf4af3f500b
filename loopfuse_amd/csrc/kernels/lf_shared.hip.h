// lf_shared.hip.h — one new token per request over keys in pages: a prefix that all requests share and each request's own
// keys, for lf_attn_decode (-DLF_SHARED=1: own keys, 2: the prefix) and lf_shared_combine.
//
// softmax over both parts splits as any softmax over splits of its keys does: each part leaves, per row, an exponent offset m,
// the sum l of the exponentials and their sum with V, and lf_shared_combine joins them.  All B * group rows of a kv head meet the
// same prefix, so its K and V are read for 16 rows (or 128) at a time instead of for every request.
//   Lengths are on the GPU only.  The own keys are cut into pieces of one length for all requests, `split`, so that about `target` workgroups
// have one, and the pieces are numbered request by request.  Every wave finds its piece by itself from the lengths (a scan of B
// numbers, 64 at a time): no launch ahead, no table, and the same numbers come out in lf_shared_combine.
#ifndef LF_SHARED_HIP_H
#define LF_SHARED_HIP_H

struct LfSharedParams : LfAttnParams {       // q_sb, q_sh, q_ss: request, kv head, row of its group; o likewise; Sk = keys of the prefix
  const int* lengths;        // [B] own keys of each request, in the pages of its row of k_table / v_table
  const void* prefix_k;      // pages of the prefix (lf_table_t)
  const void* prefix_v;
  float* pre_acc;            // [Hkv, B * rows, nsplit, D], the prefix's partials
  float* pre_ml;             // [Hkv, B * rows, nsplit, 2]
  int room;                  // own keys that a row of the tables has room for
  int units;                 // workgroups per piece of own keys
  int target;                // workgroups that the own keys are cut for
  int least;                 // least length of a piece, a multiple of 32
};                           // part_acc: [pieces, Hkv, rows, D] of own keys, part_ml: [pieces, Hkv, rows, 2]

__device__ __forceinline__ int lf_shared_length(const LfSharedParams& p, int b) {
  return b < p.B ? min(max(p.lengths[b], 0), p.room) : 0;
}
__device__ __forceinline__ int lf_shared_wave_sum(int x) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) x += __shfl_xor(x, d, 64);
  return x;
}
// length of a piece: whole pairs of 16-key steps
__device__ __forceinline__ int lf_shared_split(const LfSharedParams& p) {
  const int lane = __lane_id();
  long long total = 0;
  for (int b0 = 0; b0 < p.B; b0 += 64) total += lf_shared_wave_sum(lf_shared_length(p, b0 + lane));
  const long long even = (total * p.units + p.target - 1) / p.target;
  return __builtin_amdgcn_readfirstlane(max(p.least, (int)((even + 31) / 32 * 32)));
}
// The request of piece `piece` and its number among that request's pieces; false: there is no such piece.
__device__ __forceinline__ bool lf_shared_piece(const LfSharedParams& p, int split, int piece, int& b, int& number, int& length) {
  const int lane = __lane_id();
  int before = 0;
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    const int len = lf_shared_length(p, b0 + lane), n = (len + split - 1) / split;
    int upto = n;            // pieces of requests b0 .. b0 + lane
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int x = __shfl_up(upto, d, 64);
      if (lane >= d) upto += x;
    }
    const unsigned long long past = __builtin_amdgcn_ballot_w64(before + upto > piece);
    if (past != 0ull) {
      const int l = (int)__builtin_ctzll(past);
      b = b0 + l;
      number = piece - before - (__builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(n, l));
      length = __builtin_amdgcn_readlane(len, l);
      return true;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  return false;
}
// First piece of request `b` and how many it has.
__device__ __forceinline__ void lf_shared_pieces_of(const LfSharedParams& p, int split, int b, int& first, int& count) {
  const int lane = __lane_id();
  first = 0;
  for (int b0 = 0; b0 < b; b0 += 64) first += lf_shared_wave_sum(b0 + lane < b ? (lf_shared_length(p, b0 + lane) + split - 1) / split : 0);
  count = (lf_shared_length(p, b) + split - 1) / split;
}

#endif  // LF_SHARED_HIP_H
