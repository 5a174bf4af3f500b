// lf_paged_tables.hip — the pages of a batch of requests for their new tokens, and where each new token goes, in one launch.
//
// Request b has c = cached[b] tokens in the pages that its row of the table names and gets n = new[b] more.  With P tokens per page
//   have = ceil(c / P), need = ceil((c + n) / P) - have, first = sum of `need` of the requests before it,
//   table[b, have + i] = free[first + i], i < need,
//   offsets[b] = sum of `new` of the requests before it: the packed row of its first new token,
//   positions[offsets[b] + t] = c + t, slots[...] = table[b, (c + t) / P] * P + (c + t) % P, t < n,
//   lengths[b] = c + the number of its new tokens that fit.
// A block has one request (and a share of its tokens): it forms the two sums itself from all B lengths, which are in L2 after the first
// block, so that no block waits for another.  Slots of new pages come from the list of free ones, not from the table, so blocks of one
// request do not wait for each other's entries either.  Bound by its chain of round trips (lengths, then the page, then the stores): 64 requests of one
// new token 4.1 us, 256 of 2048 and fewer (2.2 MB) 6.1, as long as the call takes the host.
// What does not fit -- no free page left, a row of the table too short, a token behind the last row -- gets page and slot -1 and is not
// counted, so that nothing reads keys that are not there: of each kind it is the request's last tokens.

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
extern "C" __global__ void __launch_bounds__(LF_TABLES_NT) lf_paged_tables(const LfTablesParams p) {
  __shared__ long long parts[4][LF_TABLES_NT / 64];
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
  auto page_at = [&](long long i) -> lf_table_t { return i < p.count ? p.free[i] : (lf_table_t)-1; };
  const int share = blockIdx.y * LF_TABLES_NT + tid, step = gridDim.y * LF_TABLES_NT;
  if (b < p.B) {
    const long long c = cached(b), n = fresh(b), have = pages(c), need = pages(c + n) - have;
    lf_table_t* mine = p.table + b * p.table_stride;
    const long long end = min(n, p.T - row);
    if (share == 0) {
      const long long named = min((long long)p.width, have + min(need, max(p.count - first, 0ll)));      // entries of its row that name pages
      p.offsets[b] = clamp32(row);
      p.lengths[b] = clamp32(c + max(0ll, min(end, (named << p.shift) - c)));
    }
    for (long long i = share; i < need && have + i < p.width; i += step) mine[have + i] = page_at(first + i);
    for (long long t = share; t < end; t += step) {
      const long long at = (c + t) >> p.shift;
      const lf_table_t page = at >= p.width ? (lf_table_t)-1 : at < have ? mine[at] : page_at(first + at - have);
      p.positions[row + t] = clamp32(c + t);
      p.slots[row + t] = page < 0 || page > (0x7fffffff >> p.shift) ? -1 : (int)((page << p.shift) | ((c + t) & up));
    }
  }
  if (b == 0 && share == 0) {
    p.offsets[p.B] = clamp32(rows);
    p.pages[0] = clamp32(sum[3]);
  }
  // rows of no token, dealt to all blocks
  for (long long t = rows + (long long)b * step + share; t < p.T; t += (long long)gridDim.x * step) p.slots[t] = p.positions[t] = -1;
}
