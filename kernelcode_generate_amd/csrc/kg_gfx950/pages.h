// Pages and slots of a step's new tokens in the paged cache (kv_cache.h), found on the GPU from the requests' lengths, and the
// pages that a request gives back. Request b has c = context[b] cached tokens and n = added[b] new ones; its new tokens are
// the batch's rows starts[b] .. starts[b + 1] - 1, starts the running sums of n, cut where they pass the batch. Row starts[b] + i:
//   position c + i, page p = position / page_size of the request, slot = table[b, p] page_size + position % page_size.
// Free pages are a stack, `count` of them, the next one on top. New pages p of ceil(c / page_size) .. ceil((c + n) / page_size) - 1
// are taken in the order of requests and pages, the i-th of all of them free[count - 1 - i], none (-1) once the stack is empty.
// Pages that go back, of ceil(keep / page_size) .. ceil(held / page_size) - 1, are put on the stack the last one first, so that
// giving back what a call took leaves the stack as it was.
//
// A call is a chain of a few dependent reads (lengths, a search for a row's request in LDS, its page), which more workgroups do not shorten,
// and only one workgroup can take from the stack and write what is left of it without a second launch: up to 4096 rows one
// workgroup does all, more are written by a second launch. us with one launch / two, 256 requests of a token each 5.0 / 6.3, 1024 5.8 / 8.0, 4000
// 16.5 / 17.3; 6 requests in 3000 rows 6.4 / 6.5, 8 in 4096 7.3 / 6.3, 100 in 4000 8.4 / 6.8, 12 in 4800 7.9 / 6.4, 24 prompts in 16384 rows
// 19.2 / 6.6: few requests of 3000 to 4096 rows would be a microsecond or so faster with two. A launch by itself takes 2.3. Pages given back: 4.1
// for 256 entries, 4.6 for 1024; further ones go 1024 at a time, in two walks of the one workgroup: 16384 entries 36 to 41, 131072 230 to 300.
#pragma once

#include "common.h"
#include "kv_cache.h"

namespace kg_gfx950 {

constexpr int kPagesThreads = 1024;
constexpr int kPagesMostRequests = 8192;  // their sums lie in LDS

struct PagesArgs {
  long long* slots;
  int *positions, *starts, *table, *free, *count;
  const int *context, *added;  // release: keep, held
  long long slot_stride, position_stride, start_stride, table_0, table_1, free_stride, context_stride, added_stride;
  int batch, per, tokens, page_size, stack;
  PageDiv div;
};

// ceil(tokens / page_size), of pages that the table has
__device__ __forceinline__ int pages_of(int tokens, const PagesArgs& a) {
  return tokens <= 0 ? 0 : min(div_page(tokens - 1, a.div) + 1, a.per);
}

// Sums of values up to each thread's, the workgroup's total in *total; a sum is at most `most` (values are, and most < 2^31).
template <bool kCut>
__device__ __forceinline__ int pages_scan(int v, int most, int* lds, int* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  auto add = [&](int x, int y) __attribute__((always_inline)) {
    return kCut ? (int)min((uint32_t)x + (uint32_t)y, (uint32_t)most) : x + y;
  };
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int x = __shfl_up(v, o, 64);
    if (lane >= o) v = add(v, x);
  }
  __syncthreads();  // (the sums of the call before are read)
  if (lane == 63) lds[wave] = v;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kPagesThreads / 64; ++w) {
    const int x = lds[w];
    if (w < wave) before = add(before, x);
    all = add(all, x);
  }
  *total = all;
  return add(v, before);
}

// The last of sums[0 .. batch] that is at most x: a row's request, which has rows.
__device__ __forceinline__ int pages_owner(const int* sums, int batch, int x) {
  int lo = 0, hi = batch;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (sums[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Slot and position of row t, behind the sums of all requests. row_of, fresh_of: a request's first row and first of all new pages;
// context(b): its cached tokens.
template <typename F>
__device__ __forceinline__ void assign_row(const PagesArgs& a, int t, int rows, int count, const int* row_of, const int* fresh_of, F context) {
  long long slot = -1;
  int position = -1;
  if (t < rows) {
    const int b = pages_owner(row_of, a.batch, t);
    const int c = context(b);
    const uint32_t at = (uint32_t)c + (uint32_t)(t - row_of[b]);
    position = (int)min(at, 0x7fffffffu);
    if (at < 0x7fffffffu) {
      const int p = div_page(position, a.div), offset = position - p * a.page_size;
      if (p < a.per) {
        const int held = pages_of(c, a), i = fresh_of[b] + p - held;
        int* entry = a.table + b * a.table_0 + p * a.table_1;
        int old_page = -1, new_page = -1;  // (both reads on their way before either is used)
        if (p < held) old_page = *entry;
        if (p >= held && i < count) new_page = a.free[(count - 1 - i) * a.free_stride];
        const int page = p < held ? old_page : new_page;
        if (p >= held && offset == 0) *entry = page;  // (each new page's first token is one of the call's)
        if (page >= 0) slot = (long long)page * a.page_size + offset;
      }
    }
  }
  a.slots[t * a.slot_stride] = slot;
  a.positions[t * a.position_stride] = position;
}

// The requests' sums, and (kSums false) the rows. kSums: the sums go to memory for kv_assign_rows_kernel: the count of free pages as it
// was, first rows (batch + 1 of them), first new pages.
template <bool kSums>
__global__ __launch_bounds__(kPagesThreads) void kv_assign_kernel(PagesArgs a, int* sums) {
  __shared__ int row_lds[kSums ? 1 : kPagesMostRequests + 1], fresh_lds[kSums ? 1 : kPagesMostRequests],
      context_lds[kSums ? 1 : kPagesMostRequests];
  __shared__ int scan[kPagesThreads / 64], last_of[kPagesThreads / 64];
  int* row_of = kSums ? sums + 1 : row_lds;
  int* fresh_of = kSums ? sums + 2 + a.batch : fresh_lds;
  const int tid = threadIdx.x;
  const int count = max(min(*a.count, a.stack), 0);
  int rows = 0, fresh = 0;  // of the requests before
  for (int b0 = 0; b0 < a.batch; b0 += kPagesThreads) {
    const int b = b0 + tid;
    const bool real = b < a.batch;
    const int c = real ? max(a.context[b * a.context_stride], 0) : 0;
    const int n = real ? min(max(a.added[b * a.added_stride], 0), a.tokens) : 0;
    int all;
    const int upto = (int)min((uint32_t)pages_scan<true>(n, a.tokens, scan, &all) + (uint32_t)rows, (uint32_t)a.tokens);
    const int before = __shfl_up(upto, 1, 64);
    if ((tid & 63) == 63) last_of[tid >> 6] = upto;
    __syncthreads();
    const int first = (tid & 63) != 0 ? before : tid == 0 ? rows : last_of[(tid >> 6) - 1];  // (cut as the sums are)
    const int kept = upto - first;
    // tokens past 2^31 - 1 have no page
    const int end = (int)min((uint32_t)c + (uint32_t)kept, 0x7fffffffu);
    const int pages = pages_of(end, a) - pages_of(c, a);
    int new_pages;
    const int pages_upto = pages_scan<false>(pages, 0, scan, &new_pages);
    if (real) {
      row_of[b] = first;
      fresh_of[b] = fresh + pages_upto - pages;
      if (!kSums) context_lds[b] = c;
      a.starts[b * a.start_stride] = first;
    }
    rows = (int)min((uint32_t)rows + (uint32_t)all, (uint32_t)a.tokens);
    fresh += new_pages;
  }
  if (tid == 0) {
    row_of[a.batch] = rows;
    a.starts[a.batch * a.start_stride] = rows;
    if (kSums) sums[0] = count;
    *a.count = count - min(fresh, count);
  }
  if constexpr (!kSums) {
    __syncthreads();
    for (int t = tid; t < a.tokens; t += kPagesThreads) assign_row(a, t, rows, count, row_of, fresh_of, [&](int b) { return context_lds[b]; });
  }
}

__global__ __launch_bounds__(256) void kv_assign_rows_kernel(PagesArgs a, const int* sums) {
  __shared__ int row_of[kPagesMostRequests + 1];
  for (int b = threadIdx.x; b <= a.batch; b += 256) row_of[b] = sums[1 + b];
  const int count = sums[0];
  __syncthreads();
  const int rows = row_of[a.batch];
  for (long long t = (long long)blockIdx.x * 256 + threadIdx.x; t < a.tokens; t += 256ll * gridDim.x)
    assign_row(a, (int)t, rows, count, row_of, sums + 2 + a.batch, [&](int b) { return max(a.context[b * a.context_stride], 0); });
}

__global__ __launch_bounds__(kPagesThreads) void kv_release_kernel(PagesArgs a) {
  __shared__ int entry_of[kPagesMostRequests], page_of[kPagesMostRequests];  // entries of the requests before, a request's first page
  __shared__ int scan[kPagesThreads / 64];
  const int tid = threadIdx.x;
  const int count = max(min(*a.count, a.stack), 0);
  int entries = 0;
  for (int b0 = 0; b0 < a.batch; b0 += kPagesThreads) {
    const int b = b0 + tid;
    int n = 0, first = 0;
    if (b < a.batch) {
      first = pages_of(a.context[b * a.context_stride], a);
      n = max(pages_of(a.added[b * a.added_stride], a) - first, 0);
    }
    int all;
    const int upto = pages_scan<false>(n, 0, scan, &all);
    if (b < a.batch) {
      entry_of[b] = entries + upto - n;
      page_of[b] = first;
    }
    entries += all;
  }
  __syncthreads();
  auto entry = [&](int e) __attribute__((always_inline)) {
    const int b = pages_owner(entry_of, a.batch, e);
    return a.table + b * a.table_0 + (page_of[b] + e - entry_of[b]) * a.table_1;
  };
  // how many of the entries are pages: of more than a thread has one of, by a walk of its own
  const bool one = entries <= kPagesThreads;
  int pages = 0;
  if (!one) {
    int found = 0;
    for (int e = tid; e < entries; e += kPagesThreads) found += *entry(e) >= 0;
    pages_scan<false>(found, 0, scan, &pages);
  }
  int before = 0;
  for (int e0 = 0; e0 < entries; e0 += kPagesThreads) {
    const int e = e0 + tid;
    int* at = e < entries ? entry(e) : nullptr;
    const int page = at != nullptr ? *at : -1;
    int all;
    const int upto = before + pages_scan<false>(page >= 0, 0, scan, &all);
    if (one) pages = all;
    before += all;
    if (page >= 0) {
      const uint32_t spot = (uint32_t)count + (uint32_t)(pages - upto);  // (a stack of nearly 2^31 places and what goes back pass 31 bits)
      if (spot < (uint32_t)a.stack) a.free[spot * a.free_stride] = page;
    }
    if (at != nullptr) *at = -1;
  }
  if (tid == 0) *a.count = (int)min((uint32_t)count + (uint32_t)pages, (uint32_t)a.stack);
}

}  // namespace kg_gfx950
