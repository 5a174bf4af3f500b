// lf_read_kv.hip — rows of keys and values out of their slots of page pools of 16-bit rows, or of pools held in 4 bits (-DLF_READ4=1) as the
// values that they stand for: rows[t] = pool[slot[t]], zeros where there is no such slot.  A thread has 8 neighbours of a K row and the same ones of
// the V row, neighbouring threads the pieces of one row: each is a load of 16 bytes, or of 4 and a scale, and a store of 16.  Bound by memory: 10 240 rows of 8 heads of 128 out of 4 bits 11.1 us
// (53 MB, 4.8 TB/s, 3 us of it a launch's own), 64 such rows 3.1.
#ifndef LF_READ4
#define LF_READ4 0
#endif

struct LfReadParams {
  const void* k_pool;
  const void* v_pool;
  const unsigned char* k_scales;   // of pools in 4 bits
  const unsigned char* v_scales;
  lf_elem* k;                  // [T, heads, D]
  lf_elem* v;
  const int* slots;            // [T]
  long long kp_sb, kp_ss, kp_sh, vp_sb, vp_ss, vp_sh;  // pages, tokens of a page, heads (LF_READ4: bytes of a page's codes, of its scales, unused)
  long long last;              // slots of a pool
  int T, heads, per_head;      // 8-element pieces of a head's row
  int shift;                   // log2 of the tokens per page
};

extern "C" __global__ void __launch_bounds__(256) lf_read_kv(const LfReadParams p) {
  const long long piece = (long long)blockIdx.x * 256 + threadIdx.x;
  const long long row = piece / p.per_head;                 // of a token and head
  const int r8 = (int)(piece - row * p.per_head);
  const long long t = row / p.heads;
  if (t >= p.T) return;
  const int h = (int)(row - t * p.heads);
  const int slot = p.slots[t];
  lf_elem8 k = {}, v = {};
  if (slot >= 0 && slot < p.last) {
#if LF_READ4
    unsigned sk, sv;
    const unsigned ck = lf_pool4_get(false, reinterpret_cast<const unsigned char*>(p.k_pool), p.k_scales, p.kp_sb, p.kp_ss, slot, p.shift, h, r8, sk);
    const unsigned cv = lf_pool4_get(true, reinterpret_cast<const unsigned char*>(p.v_pool), p.v_scales, p.vp_sb, p.vp_ss, slot, p.shift, h, r8, sv);
    k = lf_pool4_values(ck, __builtin_bit_cast(float, sk << 23));
    v = lf_pool4_values(cv, __builtin_bit_cast(float, sv << 23));
#else
    const long long page = slot >> p.shift, at = slot & ((1 << p.shift) - 1);
    k = *reinterpret_cast<const lf_elem8*>(reinterpret_cast<const lf_elem*>(p.k_pool) + page * p.kp_sb + at * p.kp_ss + h * p.kp_sh + 8 * r8);
    v = *reinterpret_cast<const lf_elem8*>(reinterpret_cast<const lf_elem*>(p.v_pool) + page * p.vp_sb + at * p.vp_ss + h * p.vp_sh + 8 * r8);
#endif
  }
  *reinterpret_cast<lf_elem8*>(p.k + 8 * piece) = k;
  *reinterpret_cast<lf_elem8*>(p.v + 8 * piece) = v;
}
