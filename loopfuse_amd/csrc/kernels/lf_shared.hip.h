// lf_shared.hip.h — one new token per request over keys in pages: a prefix that all requests share and each request's own
// keys, for lf_attn_decode (-DLF_SHARED=1) and lf_shared_combine.
//
// softmax over both parts splits as any softmax over splits of its keys does: each part leaves, per row, an exponent offset m,
// the sum l of the exponentials and their sum with V, and lf_shared_combine joins them.  All B * group rows of a kv head meet the
// same prefix, so its K and V are read for 16 rows (or 128) at a time instead of for every request.  One launch has the workgroups of
// both: those of the prefix come first.
//   Lengths are on the GPU only.  The own keys are cut into pieces of one length for all requests, so that about 2^target_log2
// workgroups have one, and the pieces are numbered request by request.  Every wave finds its piece by itself from the lengths (a scan of
// B numbers, 64 at a time): no launch ahead, no table, and the same numbers come out in lf_shared_combine.
//   Bound by HBM where the own keys are most of it, by the chain of a split's tiles where the prefix is.  32/8 heads of 128, us of this
// launch: 64 requests up to 1024 behind 2048 keys 30 ... 34 (146 MB, 4.9 TB/s at best), 128 up to 300 behind 8208 40 (17.5 GFLOP beside 115 MB), 2 of 40 behind
// 1000 6.4.
#ifndef LF_SHARED_HIP_H
#define LF_SHARED_HIP_H

struct LfSharedParams : LfAttnParams {       // q_sb, q_sh, q_ss: request, kv head, row of its group; o likewise; Sk = keys of the prefix
  const int* lengths;        // [B] own keys of each request, in the pages of its row of k_table / v_table
  const void* prefix_k;      // pages of the prefix (lf_table_t)
  const void* prefix_v;
  float* pre_acc;            // [Hkv, nsplit, B * rows, D], the prefix's partials
  float* pre_ml;             // [Hkv, nsplit, B * rows, 2]
  int room;                  // own keys that a row of the tables has room for
  int units;                 // workgroups per piece of own keys
  int pre_units;             // workgroups per split of the prefix ...
  int pre_blocks;            // ... and in all
  int target_log2;           // workgroups that the own keys are cut for
  int least;                 // least length of a piece, a multiple of 32
};                           // part_acc: [pieces, Hkv, rows, D] of own keys, part_ml: [pieces, Hkv, rows, 2]

__device__ __forceinline__ int lf_shared_length(const LfSharedParams& p, int b) {
  return b < p.B ? min(max(p.lengths[b], 0), p.room) : 0;
}
// sum of x over lanes 0 ... this one: within rows of 16 lanes, then across them
__device__ __forceinline__ int lf_wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);      // row_shr:1, 2, 4, 8
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);      // row_bcast:15 into rows 1 and 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);      // row_bcast:31 into rows 2 and 3
  return x;
}
// length of a piece: whole pairs of 16-key steps.  `mine` = lengths of the first 64 requests, one per lane (read once for all scans)
__device__ __forceinline__ int lf_shared_split(const LfSharedParams& p, int mine) {
  const int lane = __lane_id();
  long long total = 0;
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    const int len = b0 ? lf_shared_length(p, b0 + lane) : mine;
    // (the sum of 64 lengths may not fit 32 bits: their halves do)
    total += (long long)__builtin_amdgcn_readlane(lf_wave_scan(len >> 16), 63) << 16;
    total += __builtin_amdgcn_readlane(lf_wave_scan(len & 0xffff), 63);
  }
  const long long even = (total * p.units) >> p.target_log2;
  return max(p.least, (int)min((even + 32) & ~31ll, 1ll << 30));
}
// The request of piece `piece`, the piece's number among that request's and the request's keys; false: there is no such piece.
__device__ __forceinline__ bool lf_shared_piece(const LfSharedParams& p, int mine, int split, int piece, int& b, int& number, int& keys) {
  const int lane = __lane_id();
  int before = 0;
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    const int len = b0 ? lf_shared_length(p, b0 + lane) : mine, n = (len + split - 1) / split;
    const int upto = lf_wave_scan(n);            // pieces of requests b0 .. b0 + lane
    const unsigned long long past = __builtin_amdgcn_ballot_w64(before + upto > piece);
    if (past != 0ull) {
      const int l = (int)__builtin_ctzll(past);
      b = b0 + l;
      number = piece - before - (__builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(n, l));
      keys = __builtin_amdgcn_readlane(len, l);
      return true;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  return false;
}
// First piece of request `b` and how many it has.
__device__ __forceinline__ void lf_shared_pieces_of(const LfSharedParams& p, int mine, int split, int b, int& first, int& count) {
  const int lane = __lane_id();
  first = count = 0;
  for (int b0 = 0; b0 <= b; b0 += 64) {
    const int n = ((b0 ? lf_shared_length(p, b0 + lane) : mine) + split - 1) / split;
    first += __builtin_amdgcn_readlane(lf_wave_scan(b0 + lane < b ? n : 0), 63);
    if (b - b0 < 64) count = __builtin_amdgcn_readlane(n, b - b0);
  }
}

// What a workgroup of lf_attn_decode does: a split of the prefix for 16 rows of all requests, or a piece of one request's own keys.
struct LfSharedUnit {
  bool prefix;
  int b;                     // request (prefix: 0)
  int z;                     // split, or piece among its request's
  int piece;                 // piece among all
  int keys, split_len;       // keys of the prefix or the request, and of a split or piece
  int unit;                  // (kv head or heads, chunk of rows) of it
  int rows;                  // query rows per kv head: of all requests, or of one
  const void* k_table;
  const void* v_table;
};
__device__ __forceinline__ bool lf_shared_unit(const LfSharedParams& p, int block, LfSharedUnit& u) {
#if !LF_PREFIX               /* (else the workgroups of the prefix went to lf_prefix_tile) */
  if (block < p.pre_blocks) {
    u = LfSharedUnit{true, 0, block / p.pre_units, 0, p.Sk, p.split_len, block % p.pre_units, p.B * p.rows, p.prefix_k, p.prefix_v};
    return true;
  }
#endif
  block -= p.pre_blocks;
  const int mine = lf_shared_length(p, __lane_id());
  const int split = lf_shared_split(p, mine), piece = block / p.units;
  int b, z, keys;
  if (!lf_shared_piece(p, mine, split, piece, b, z, keys)) return false;
  u = LfSharedUnit{false, __builtin_amdgcn_readfirstlane(b), __builtin_amdgcn_readfirstlane(z), piece, __builtin_amdgcn_readfirstlane(keys),
                   __builtin_amdgcn_readfirstlane(split), block - piece * p.units, p.rows, p.k_table, p.v_table};
  return true;
}

#endif  // LF_SHARED_HIP_H
