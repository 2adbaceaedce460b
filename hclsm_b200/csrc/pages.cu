// Page tables of a paged state cache: how many pages each entry's tokens need, kept on the device so that lengths never
// come to the host.  All work is a prefix sum over the entries and a move of page numbers; the bound is the latency
// of a handful of dependent loads (resize) and the slots written (slots).
//
// Released pages have ranks 0 ... R - 1 (entries, then places ascending), wanted places ranks 0 ... W - 1.  Pushed with the
// first on top and then popped, the released page of rank r goes to the wanted place of rank r where r < W, else to place
// n + R - 1 - r of the stack; a wanted place of rank w >= R gets what lay at n - 1 - (w - R).  So, once the request is
// known to be valid, the pages can move in any order.
#include <cooperative_groups.h>

#include "common.cuh"

namespace hclsm {
int* device_err_ptr();
int num_sms();

namespace pages {

constexpr int kThreads = 1024, kFewThreads = 256, kCluster = 8;

struct Resize {
  int32_t *table, *stack, *n_free;
  const int32_t *old_lens, *new_lens;
  int B, M, P, shift;
  int* err;
};

// Exclusive sums of (released, wanted) over the block's threads; total: the block's.
__device__ __forceinline__ int2 scan(int2 v, int2* warp_sum, int2& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  int2 s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, s.x, o), y = __shfl_up_sync(0xffffffffu, s.y, o);
    if (lane >= o) s.x += x, s.y += y;
  }
  __syncthreads();
  if (lane == 31) warp_sum[warp] = s;
  __syncthreads();
  int2 w = lane < warps ? warp_sum[lane] : make_int2(0, 0);
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, w.x, o), y = __shfl_up_sync(0xffffffffu, w.y, o);
    if (lane >= o) w.x += x, w.y += y;
  }
  total = make_int2(__shfl_sync(0xffffffffu, w.x, 31), __shfl_sync(0xffffffffu, w.y, 31));
  const int before = max(warp - 1, 0);
  const int x = __shfl_sync(0xffffffffu, w.x, before), y = __shfl_sync(0xffffffffu, w.y, before);
  return make_int2((warp ? x : 0) + s.x - v.x, (warp ? y : 0) + s.y - v.y);
}

// The entry with the i-th released or wanted page: the last one that begins at or before it.
template <bool WANTED> __device__ __forceinline__ int entry_of(const int2* off, int entries, int i) {
  int lo = 0;
#pragma unroll
  for (int step = kThreads / 2; step > 0; step >>= 1)
    if (lo + step < entries && (WANTED ? off[lo + step].y : off[lo + step].x) <= i) lo += step;
  return lo;
}

// One cluster (of one block where the table is small).  Each block forms all the sums, since entries are few next to
// their pages; the pages are shared out among all threads by their place in the order, so entries of any size cost
// the same.  Pages of an order's run: a search in the sums of up to a block's threads of entries.
__global__ void __launch_bounds__(kThreads) resize_kernel(const __grid_constant__ Resize p) {
  namespace cg = cooperative_groups;
  __shared__ int2 warp_sum[kThreads / 32], off[kThreads + 1];
  __shared__ int2 span[kThreads];  // pages an entry had, has
  __shared__ int bad, many;
  pdl_wait();
  pdl_trigger();
  const cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, nt = blockDim.x;
  const int me = (int)cluster.block_rank() * nt + tid, all = (int)cluster.num_blocks() * nt;
  if (tid == 0) bad = many = 0;
  __syncthreads();
  const int n = *p.n_free;
  const int64_t most = (int64_t)p.M << p.shift;
  // pass 0 counts and checks, 1 releases, 2 takes
  int64_t released = 0, wanted = 0;  // over all entries
  for (int pass = 0; pass < 3; ++pass) {
    if (pass == 1 && released == 0) continue;
    if (pass == 2 && wanted == 0) continue;
    int2 done = make_int2(0, 0);
    for (int b0 = 0; b0 < p.B; b0 += nt) {
      const int b = b0 + tid, entries = min(nt, p.B - b0);
      int32_t first = -1;  // what this thread's entry has at the first place that it wants: asked for before the sums
      if (pass == 0 || p.B > nt) {  // one round of entries stays where it is
        int2 s = make_int2(0, 0);
        if (b < p.B) {
          const int from = p.old_lens[b], to = p.new_lens[b];
          if (from < 0 || to < 0 || from > most || to > most)
            bad = 1;
          else
            s = make_int2((int)(((int64_t)from + (1 << p.shift) - 1) >> p.shift),
                          (int)(((int64_t)to + (1 << p.shift) - 1) >> p.shift));
          if (pass == 0 && s.y > s.x) {
            first = p.table[(int64_t)b * p.M + s.x];
            if (s.y > s.x + 1) many = 1;
          }
        }
        int2 total;
        const int2 at = scan(make_int2(max(s.x - s.y, 0), max(s.y - s.x, 0)), warp_sum, total);
        span[tid] = s;
        off[tid] = at;  // behind the last entry: the total
        if (tid == 0) off[nt] = total;
        __syncthreads();
      }
      const int2 total = off[entries];
      // the pages of these entries, in order
      const int count = pass == 2 ? total.y : total.x;
      // four pages at a time: a thread waits for memory once for them
      for (int i0 = me; i0 < count; i0 += 4 * all) {
        int32_t* at[4];
        int32_t page[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = i0 + e * all;
          at[e] = nullptr;
          if (i >= count) continue;
          const int lo = pass == 2 ? entry_of<true>(off, entries, i) : entry_of<false>(off, entries, i);
          at[e] = p.table + (int64_t)(b0 + lo) * p.M + (pass == 2 ? span[lo].x + i - off[lo].y : span[lo].y + i - off[lo].x);
          page[e] = pass == 2 ? p.stack[n + (int)released - 1 - (done.y + i)] : *at[e];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (!at[e]) continue;
          const int i = i0 + e * all;
          if (pass == 0) {
            if ((unsigned)page[e] >= (unsigned)p.P) bad = 1;
          } else if (pass == 1) {
            p.stack[n + (int)released - 1 - (done.x + i)] = page[e];
            *at[e] = -1;
          } else {
            *at[e] = page[e];
            p.stack[n + (int)released - 1 - (done.y + i)] = -1;
          }
        }
      }
      if (pass == 0) {  // a wanted place that holds a page: the page would be lost
        if (first >= 0) bad = 1;
        if (many) {
#pragma unroll 4
          for (int i = me; i < total.y; i += all) {
            const int lo = entry_of<true>(off, entries, i);
            if (p.table[(int64_t)(b0 + lo) * p.M + span[lo].x + i - off[lo].y] >= 0) bad = 1;
          }
        }
      }
      done.x += total.x, done.y += total.y;
      if (p.B > nt) __syncthreads();
    }
    if (pass == 0) {
      released = done.x, wanted = done.y;
      if (n < 0 || n > p.P || n + released > p.P || wanted > n + released) {
        if (tid == 0) bad = 1;
      } else {  // the pages that were on the stack before and are taken now
#pragma unroll 8
        for (int i = me; i < (int)(wanted - released); i += all)
          if ((unsigned)p.stack[n - 1 - i] >= (unsigned)p.P) bad = 1;
      }
      cluster.sync();  // the checks before the first change
      int any = 0;
      for (int r = 0; r < (int)cluster.num_blocks(); ++r) any |= *cluster.map_shared_rank(&bad, r);
      cluster.sync();  // no block leaves while others read its flag
      if (any) {
        if (me == 0) record_error(p.err, HCLSM_ERR_SHAPE);
        return;
      }
    } else {
      cluster.sync();  // the releases before the first taking
    }
  }
  if (me == 0) *p.n_free = n + (int)(released - wanted);
}

// ---- large tables: a kernel that checks and one that moves, over all SMs ---------------------------------
// Up to kThreads entries.  131072 pages: 6 to 7 us in the two, 22 in one cluster.
constexpr int kBlocks = 128;

struct Round {
  int2 off[kThreads + 1];  // released and wanted pages before an entry; behind the last: of all
  int2 span[kThreads];     // pages an entry had, has
  int2 warp_sum[kThreads / 32];
};

// The entries; false where a length lies outside the table.
__device__ __forceinline__ bool load(const Resize& p, Round& r) {
  const int b = threadIdx.x;
  const int64_t most = (int64_t)p.M << p.shift;
  int2 s = make_int2(0, 0);
  bool fine = true;
  if (b < p.B) {
    const int from = p.old_lens[b], to = p.new_lens[b];
    fine = from >= 0 && to >= 0 && from <= most && to <= most;
    if (fine)
      s = make_int2((int)(((int64_t)from + (1 << p.shift) - 1) >> p.shift),
                    (int)(((int64_t)to + (1 << p.shift) - 1) >> p.shift));
  }
  int2 total;
  const int2 at = scan(make_int2(max(s.x - s.y, 0), max(s.y - s.x, 0)), r.warp_sum, total);
  r.span[b] = s;
  r.off[b] = at;
  if (b == 0) r.off[kThreads] = total;
  __syncthreads();
  return fine;
}
// The place in the table of the i-th released or wanted page.
template <bool WANTED> __device__ __forceinline__ int32_t* place(const Resize& p, const Round& r, int i) {
  const int lo = entry_of<WANTED>(r.off, p.B, i);
  return p.table + (int64_t)lo * p.M + (WANTED ? r.span[lo].x + i - r.off[lo].y : r.span[lo].y + i - r.off[lo].x);
}

// ws: whether each block found a fault, then the free pages.
__global__ void __launch_bounds__(kThreads) check_kernel(const __grid_constant__ Resize p, int32_t* ws) {
  __shared__ Round r;
  pdl_wait();
  pdl_trigger();
  const int me = blockIdx.x * kThreads + threadIdx.x, all = gridDim.x * kThreads;
  const int n = *p.n_free;
  bool fine = load(p, r);
  const int R = r.off[kThreads].x, W = r.off[kThreads].y;
  fine = fine && n >= 0 && n <= p.P && (int64_t)n + R <= p.P && W <= (int64_t)n + R;
  if (__syncthreads_and(fine)) {  // else the places below may not exist
    for (int i = me; i < R; i += all) fine = fine && (unsigned)*place<false>(p, r, i) < (unsigned)p.P;
    for (int i = me; i < W; i += all) fine = fine && *place<true>(p, r, i) < 0;  // a page there would be lost
    for (int i = me; i < W - R; i += all) fine = fine && (unsigned)p.stack[n - 1 - i] < (unsigned)p.P;
  }
  const int all_fine = __syncthreads_and(fine);
  if (threadIdx.x == 0) ws[blockIdx.x] = !all_fine;
  if (me == 0) ws[gridDim.x] = n;
}

__global__ void __launch_bounds__(kThreads) move_kernel(const __grid_constant__ Resize p, const int32_t* ws) {
  __shared__ Round r;
  pdl_wait();
  pdl_trigger();
  const int me = blockIdx.x * kThreads + threadIdx.x, all = gridDim.x * kThreads;
  const int n = ws[gridDim.x];
  if (__syncthreads_or((int)threadIdx.x < (int)gridDim.x && ws[threadIdx.x])) {
    if (me == 0) record_error(p.err, HCLSM_ERR_SHAPE);
    return;
  }
  load(p, r);
  const int R = r.off[kThreads].x, W = r.off[kThreads].y;
  for (int i = me; i < W; i += all) {
    int32_t* from = i < R ? place<false>(p, r, i) : p.stack + (n - 1 - (i - R));
    const int32_t page = *from;
    *from = -1;
    *place<true>(p, r, i) = page;
    if (i < R) p.stack[n + R - 1 - i] = -1;
  }
  for (int i = W + me; i < R; i += all) {
    int32_t* from = place<false>(p, r, i);
    p.stack[n + R - 1 - i] = *from;
    *from = -1;
  }
  if (me == 0) *p.n_free = n + R - W;
}

struct Slots {
  const int32_t *table, *start, *count;
  int32_t* slots;
  int B, M, n, shift;
};

// Four slots a thread, blockIdx.y the entry; `wide`: a row of slots is whole 16 bytes.
__global__ void __launch_bounds__(256) slots_kernel(const __grid_constant__ Slots p, int wide) {
  pdl_wait();
  pdl_trigger();
  const uint32_t mask = (1u << p.shift) - 1;
  const int64_t most = (int64_t)p.M << p.shift;
  for (int b = blockIdx.y; b < p.B; b += gridDim.y) {
    const int32_t* row = p.table + (int64_t)b * p.M;
    int32_t* out = p.slots + (int64_t)b * p.n;
    const int64_t start = p.start[b];
    const int count = p.count ? min(p.count[b], p.n) : p.n;
    for (int64_t j = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; j < p.n; j += (int64_t)gridDim.x * 1024) {
      int s[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t at = start + j + e;
        s[e] = -1;
        if (j + e < count && at >= 0 && at < most) {
          const int page = row[at >> p.shift];
          // a number that no slot of 31 bits holds: the last slot, which is behind every cache
          if (page >= 0) s[e] = page >> (31 - p.shift) ? 0x7fffffff : (int)((uint32_t)page << p.shift | ((uint32_t)at & mask));
        }
      }
      if (wide) {
        *reinterpret_cast<int4*>(out + j) = make_int4(s[0], s[1], s[2], s[3]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (j + e < p.n) out[j + e] = s[e];
      }
    }
  }
}

bool power_of_2(int n) { return n > 0 && (n & (n - 1)) == 0; }
int log2_of(int n) {
  int l = 0;
  while (n >> 1) n >>= 1, ++l;
  return l;
}

}  // namespace pages
}  // namespace hclsm

using namespace hclsm;

// Where the two kernels over all SMs pay: more pages than a cluster moves in a few microseconds.
static bool wide(int32_t B, int32_t M) { return B <= pages::kThreads && (int64_t)B * M > 16384; }

extern "C" size_t hclsm_pages_resize_workspace_size(int32_t B, int32_t M) {
  return B > 0 && M > 0 && wide(B, M) ? (pages::kBlocks + 1) * sizeof(int32_t) : 0;
}

extern "C" int hclsm_pages_resize(int32_t* table, int32_t B, int32_t M, int32_t* stack, int32_t* n_free, int32_t P,
                                  int32_t page, const int32_t* old_lens, const int32_t* new_lens, void* ws,
                                  size_t ws_bytes, void* stream) {
  if (B < 0 || M < 0 || P < 0 || !pages::power_of_2(page)) return HCLSM_ERR_SHAPE;
  // the kernels' indices go past the last page by their stride, at most 2^18
  if ((int64_t)P * page > 0x7fffffff || (int64_t)B * M > 0x7fffffff - (1 << 18)) return HCLSM_ERR_SHAPE;
  if (B == 0) return HCLSM_OK;
  if ((!table && M) || (!stack && P) || !n_free || !old_lens || !new_lens) return HCLSM_ERR_NULL;
  const size_t need = hclsm_pages_resize_workspace_size(B, M);
  if (ws_bytes < need || (need && !ws)) return HCLSM_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(ws) % 16) return HCLSM_ERR_ALIGN;
  pages::Resize p = {table, stack, n_free, old_lens, new_lens, B, M, P, pages::log2_of(page), device_err_ptr()};
  if (need) {
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    int32_t* flags = static_cast<int32_t*>(ws);
    if (const int rc = launch_pdl(pages::check_kernel, pages::kBlocks, pages::kThreads, 0, st, p, flags)) return rc;
    return launch_pdl(pages::move_kernel, pages::kBlocks, pages::kThreads, 0, st, p, flags);
  }
  // one small block takes a table of a few thousand pages faster than a cluster meets at its barriers
  const bool few = (int64_t)B * M <= 8192 && B <= pages::kFewThreads;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = few ? 1 : pages::kCluster, cfg.blockDim = few ? pages::kFewThreads : pages::kThreads;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = few ? 1 : pages::kCluster, attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr, cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, pages::resize_kernel, p) == cudaSuccess ? HCLSM_OK : HCLSM_ERR_LAUNCH;
}

extern "C" int hclsm_page_slots(const int32_t* table, int32_t B, int32_t M, int32_t page, const int32_t* start,
                                const int32_t* count, int32_t n, int32_t* slots, void* stream) {
  if (B < 0 || M < 0 || n < 0 || !pages::power_of_2(page)) return HCLSM_ERR_SHAPE;
  const int64_t total = (int64_t)B * n;
  if (total == 0) return HCLSM_OK;
  if ((!table && M) || !start || !slots) return HCLSM_ERR_NULL;
  pages::Slots p = {table, start, count, slots, B, M, n, pages::log2_of(page)};
  const int64_t blocks = ((int64_t)n + 1023) / 1024, most = (int64_t)num_sms() * 8 / B + 1;
  const int wide = n % 4 == 0 && reinterpret_cast<uintptr_t>(slots) % 16 == 0;
  return launch_pdl(pages::slots_kernel, dim3((unsigned)(blocks < most ? blocks : most), (unsigned)(B < 65535 ? B : 65535)), 256, 0,
                    static_cast<cudaStream_t>(stream), p, wide);
}
