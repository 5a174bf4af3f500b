// lf_pool4.hip.h — page pools that hold keys or values in 4 bits: where their codes lie, and how rows become codes.
//
// A value is a code (bit 3 the sign, bits 0 ... 2 one of 0 0.5 1 1.5 2 3 4 6) times 2^(scale - 127), the scale a byte that 32 neighbours of a row
// share, 255 for NaN.  A pool has, page by page, its heads, each with its tokens in tiles of 16: 8 D bytes of codes and D / 2 of scales a tile.
// Within a tile the codes lie as the wave reads them that takes the tile, 64 threads (c = lane % 16, g = lane / 16):
//   keys   : row after row, D / 2 bytes of token c; two neighbours to a byte, the first in its lower half.  Thread (c, g) reads elements D / 4 * g ... of
//            token c at once, 8 bytes at D 64 and 16 at 128, which share a scale.  Scales: [token][block].
//   values : [token / 4][c][token % 4][D / 32 bytes], the bytes being elements D / 16 * c ... of the token.  Thread (c, g) reads its elements of tokens
//            4 g ... 4 g + 3 at once, as many bytes: a column of the transposed operand.  Scales: [token / 4][block][token % 4].
#ifndef LF_POOL4_HIP_H
#define LF_POOL4_HIP_H

// Codes of 8 neighbours of a row, of which four threads next to each other have 32, and the scale of those.
__device__ __forceinline__ unsigned lf_pool4_codes(const lf_elem8& y, unsigned& scale) {
  constexpr unsigned kMost = LF_DTYPE == 0 ? 252 : 140;      // 6 * 2^125, 6 * 2^13: the next power's 4 is beyond the type
  float x[8];
  unsigned top = 0;                                          // largest size by its bits, NaN beyond infinity
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = lf_to_float(y[i]);
    top = max(top, __builtin_bit_cast(unsigned, x[i]) & 0x7fffffffu);
  }
  top = max(top, (unsigned)__builtin_amdgcn_update_dpp(0, (int)top, 0xb1, 0xf, 0xf, false));       // quad_perm [1,0,3,2]
  top = max(top, (unsigned)__builtin_amdgcn_update_dpp(0, (int)top, 0x4e, 0xf, 0xf, false));       // quad_perm [2,3,0,1]
  const int e = (int)(top >> 23) - 2 + ((top & 0x7fffffu) >= 0x600000u ? 1 : 0);
  scale = top >= 0x7f800000u ? 255u : (unsigned)min(max(e, 0), (int)kMost);
  const float by = __builtin_bit_cast(float, scale == 255u ? 0x3f800000u : scale << 23);
  unsigned codes = 0;
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[0], x[1], by, 0);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[2], x[3], by, 1);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[4], x[5], by, 2);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[6], x[7], by, 3);
  return codes;
}

// Where 8 neighbours from 8 r8 of a head's row of a token lie, and their scale.
__device__ __forceinline__ long long lf_pool4_tile(long long sb, int slot, int shift, int head, int bytes) {
  const int in = slot & ((1 << shift) - 1);
  return (long long)(slot >> shift) * sb + (((long long)head << (shift - 4)) + (in >> 4)) * bytes;
}
// (of values at D 64 two neighbouring threads' elements lie in two places of 2 bytes each)
__device__ __forceinline__ void lf_pool4_put(bool values, unsigned char* codes_of, unsigned char* scales_of, long long codes_sb, long long scales_sb, int slot, int shift, int head, int r8,
                                             unsigned codes, unsigned scale) {
  constexpr int kD = LF_HEAD_DIM;
  unsigned char* tile = codes_of + lf_pool4_tile(codes_sb, slot, shift, head, 8 * kD);
  unsigned char* scales = scales_of + lf_pool4_tile(scales_sb, slot, shift, head, kD / 2);
  const int tok = slot & 15, g = tok >> 2, u = tok & 3;
  if (!values) {
    *reinterpret_cast<unsigned*>(tile + tok * (kD / 2) + 4 * r8) = codes;
    if (r8 % 4 == 0) scales[tok * (kD / 32) + r8 / 4] = (unsigned char)scale;
  } else {
    if (kD == 128) {
      *reinterpret_cast<unsigned*>(tile + ((g * 16 + r8) * 4 + u) * 4) = codes;
    } else {
      *reinterpret_cast<unsigned short*>(tile + ((g * 16 + 2 * r8) * 4 + u) * 2) = (unsigned short)codes;
      *reinterpret_cast<unsigned short*>(tile + ((g * 16 + 2 * r8 + 1) * 4 + u) * 2) = (unsigned short)(codes >> 16);
    }
    if (r8 % 4 == 0) scales[(g * (kD / 32) + r8 / 4) * 4 + u] = (unsigned char)scale;
  }
}
__device__ __forceinline__ unsigned lf_pool4_get(bool values, const unsigned char* codes_of, const unsigned char* scales_of, long long codes_sb, long long scales_sb, int slot, int shift,
                                                 int head, int r8, unsigned& scale) {
  constexpr int kD = LF_HEAD_DIM;
  const unsigned char* tile = codes_of + lf_pool4_tile(codes_sb, slot, shift, head, 8 * kD);
  const unsigned char* scales = scales_of + lf_pool4_tile(scales_sb, slot, shift, head, kD / 2);
  const int tok = slot & 15, g = tok >> 2, u = tok & 3;
  scale = values ? scales[(g * (kD / 32) + r8 / 4) * 4 + u] : scales[tok * (kD / 32) + r8 / 4];
  if (!values) return *reinterpret_cast<const unsigned*>(tile + tok * (kD / 2) + 4 * r8);
  if (kD == 128) return *reinterpret_cast<const unsigned*>(tile + ((g * 16 + r8) * 4 + u) * 4);
  return *reinterpret_cast<const unsigned short*>(tile + ((g * 16 + 2 * r8) * 4 + u) * 2) |
         (unsigned)*reinterpret_cast<const unsigned short*>(tile + ((g * 16 + 2 * r8 + 1) * 4 + u) * 2) << 16;
}

// Two values of byte `m` of 8 codes, times a power of two.
typedef lf_elem lf_pool4_two __attribute__((ext_vector_type(2)));
template <int m>
__device__ __forceinline__ lf_pool4_two lf_pool4_pair(unsigned codes, float by) {
#if LF_DTYPE == 0
  return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, by, m);
#else
  return __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, by, m);
#endif
}
__device__ __forceinline__ lf_elem8 lf_pool4_values(unsigned codes, float by) {
  const lf_pool4_two a = lf_pool4_pair<0>(codes, by), b = lf_pool4_pair<1>(codes, by), c = lf_pool4_pair<2>(codes, by), d = lf_pool4_pair<3>(codes, by);
  return lf_elem8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

#endif  // LF_POOL4_HIP_H
