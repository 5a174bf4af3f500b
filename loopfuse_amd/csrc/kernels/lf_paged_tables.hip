// lf_paged_tables.hip — the pages of a batch of requests for their new tokens, and where each new token goes, in one launch.
//
// Request b has c = cached[b] tokens in the pages that its row of the table names and gets n = new[b] more.  With P tokens per page
//   have = ceil(c / P), need = ceil((c + n) / P) - have, first = sum of `need` of the requests before it,
//   table[b, have + i] = free[first + i], i < need,
//   offsets[b] = sum of `new` of the requests before it: the packed row of its first new token,
//   positions[offsets[b] + t] = c + t, slots[...] = table[b, (c + t) / P] * P + (c + t) % P, t < n,
//   lengths[b] = c + the number of its new tokens in front of the first that has no slot.
// A block has one request (and a share of its tokens): it forms the two sums itself from all B lengths, which are in L2 after the first
// block, so that no block waits for another.  Slots of new pages come from the list of free ones, not from the table, so blocks of one
// request do not wait for each other's entries either.  The first of them looks for the first page that is none.  Bound by its chain of
// round trips (lengths, then the pages, then the stores): 64 requests of one new token 4.4 us, 256 of 2048 and fewer (2.2 MB) 6.4, as long as the
// call takes the host.
// What does not fit -- no free page left, a row of the table too short, a token behind the last row -- gets page and slot -1.  A page id below 0 or
// whose slots are no numbers in 32 bits is no page either: its tokens get slot -1.  lengths[b] ends in front of the first token without a slot,
// so that nothing reads keys that are not there.

struct LfTablesParams {
  const int* cached;          // [B]
  const int* fresh;           // [B] new tokens
  lf_table_t* table;          // [B, width], rows table_stride apart
  const lf_table_t* free;     // [count]
  int* offsets;               // [B + 1]
  int* lengths;               // [B]
  int* slots;                 // [T]
  int* positions;             // [T]
  int* pages;                 // [1] pages that the requests need
  long long table_stride;
  int B, width, count, T;
  int shift;                  // log2 of the tokens per page
};

#define LF_TABLES_NT 256
#define LF_TABLES_LOOK 8
#if LF_TABLE_I64
typedef unsigned long long lf_page_id;
#else
typedef unsigned lf_page_id;
#endif
struct LfFourIds {           // anywhere in a list
  lf_page_id id[4];
};
extern "C" __global__ void __launch_bounds__(LF_TABLES_NT) lf_paged_tables(const LfTablesParams p) {
  __shared__ long long parts[4][LF_TABLES_NT / 64];
  __shared__ int nones[LF_TABLES_NT / 64];
  const int tid = threadIdx.x, b = blockIdx.x, up = (1 << p.shift) - 1;
  auto cached = [&](int j) -> long long { return max(p.cached[j], 0); };
  auto fresh = [&](int j) -> long long { return max(p.fresh[j], 0); };
  auto pages = [&](long long tokens) { return (tokens + up) >> p.shift; };
  long long sum[4] = {0, 0, 0, 0};          // tokens before, in all; pages before, in all
  for (int j = tid; j < p.B; j += LF_TABLES_NT) {
    const long long c = cached(j), n = fresh(j), need = pages(c + n) - pages(c);
    sum[1] += n;
    sum[3] += need;
    if (j < b) {
      sum[0] += n;
      sum[2] += need;
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) sum[i] += __shfl_xor(sum[i], d, 64);
    if (tid % 64 == 0) parts[i][tid / 64] = sum[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    sum[i] = 0;
#pragma unroll
    for (int w = 0; w < LF_TABLES_NT / 64; ++w) sum[i] += parts[i][w];
  }
  const long long row = sum[0], rows = sum[1], first = sum[2];
  auto clamp32 = [](long long x) { return (int)min(x, 0x7fffffffll); };
  const int share = blockIdx.y * LF_TABLES_NT + tid, step = gridDim.y * LF_TABLES_NT;
  if (b < p.B) {
    const long long c = cached(b), n = fresh(b), have = pages(c), need = pages(c + n) - have;
    lf_table_t* mine = p.table + b * p.table_stride;
    const long long end = min(n, p.T - row);      // new tokens that have a row
    auto new_page = [&](long long i) -> lf_table_t { return first + i < p.count ? p.free[first + i] : (lf_table_t)-1; };
    // the page of entry `at` if a slot of it is a number in 32 bits, else -1
    auto page_at = [&](long long at) -> lf_table_t {
      const lf_table_t page = at >= p.width ? (lf_table_t)-1 : at < have ? mine[at] : new_page(at - have);
      return page > (0x7fffffff >> p.shift) ? (lf_table_t)-1 : page;
    };
    if (blockIdx.y == 0) {
      // The first of the new tokens' pages that is none ends the request: a page that it has begun (one at most), then new ones, neighbours in the list.
      // Those that there are no ids for are known without a look.
      const long long from = c >> p.shift;
      const int count = end > 0 ? (int)(((c + end - 1) >> p.shift) - from) + 1 : 0, begun = count > 0 && from < have, fresh_ones = count - begun;
      const int ids = (int)max(0ll, min((long long)fresh_ones, min(p.width - have, p.count - first)));
      int none = begun && page_at(from) < 0 ? 0 : ids < fresh_ones ? begun + ids : count;
      const lf_table_t* list = p.free + first;
      const lf_page_id most = 0x7fffffff >> p.shift;      // (a negative id is beyond it as an unsigned one)
      if (ids > 64) {
        // whether there is one at all: the largest id, by loads of four ids of which a thread has LF_TABLES_LOOK under way.  20 000 one-token pages of
        // one request, us, a page at a time 19.8, eight 11.4, so 6.5, without the look 5.1; 500 pages each of 16 requests 5.5, 5.9, 5.8, 4.8
        lf_page_id top = 0;
        for (unsigned i = 4 * tid; i < (unsigned)ids; i += LF_TABLES_LOOK * 4 * LF_TABLES_NT) {
          LfFourIds four[LF_TABLES_LOOK];
#pragma unroll
          for (int u = 0; u < LF_TABLES_LOOK; ++u)
            four[u] = *reinterpret_cast<const LfFourIds*>(list + min(i + u * 4 * LF_TABLES_NT, (unsigned)ids - 4));
#pragma unroll
          for (int u = 0; u < LF_TABLES_LOOK; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) top = max(top, four[u].id[e]);
        }
        if (__syncthreads_or(top > most)) {
          for (unsigned i = tid; i < (unsigned)ids; i += LF_TABLES_NT)
            if ((lf_page_id)list[i] > most) none = min(none, begun + (int)i);
#pragma unroll
          for (int d = 1; d < 64; d <<= 1) none = min(none, __shfl_xor(none, d, 64));
          if (tid % 64 == 0) nones[tid / 64] = none;
          __syncthreads();
#pragma unroll
          for (int w = 0; w < LF_TABLES_NT / 64; ++w) none = min(none, nones[w]);
        }
      } else if (ids > 0 && tid < 64) {
        // ... of few, the first one by a wave alone: 64 requests of one new token 4.2 us, by all with a barrier 4.3, without the look 3.9
        const unsigned long long bad = __builtin_amdgcn_ballot_w64(tid < ids && (lf_page_id)list[min(tid, ids - 1)] > most);
        if (bad != 0ull) none = min(none, begun + (int)__builtin_ctzll(bad));
      }
      if (tid == 0) {
        p.offsets[b] = clamp32(row);
        p.lengths[b] = clamp32(c + max(0ll, none < count ? ((from + none) << p.shift) - c : end));
      }
    }
    for (long long i = share; i < need && have + i < p.width; i += step) mine[have + i] = new_page(i);
    for (long long t = share; t < end; t += step) {
      const lf_table_t page = page_at((c + t) >> p.shift);
      p.positions[row + t] = clamp32(c + t);
      p.slots[row + t] = page < 0 ? -1 : (int)((page << p.shift) | ((c + t) & up));
    }
  }
  if (b == 0 && share == 0) {
    p.offsets[p.B] = clamp32(rows);
    p.pages[0] = clamp32(sum[3]);
  }
  // rows of no token, dealt to all blocks
  for (long long t = rows + (long long)b * step + share; t < p.T; t += (long long)gridDim.x * step) p.slots[t] = p.positions[t] = -1;
}
