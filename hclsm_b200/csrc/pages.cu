// Page tables of a paged state cache: how many pages each entry's tokens need, kept on the device so that lengths never
// come to the host.  All work is a prefix sum over the entries and a move of page numbers; the bound is the latency
// of a handful of dependent loads (resize) and the slots written (slots).
#include <cooperative_groups.h>

#include "common.cuh"

namespace hclsm {
int* device_err_ptr();
int num_sms();

namespace pages {

constexpr int kThreads = 1024, kWarps = kThreads / 32, kCluster = 8;

struct Resize {
  int32_t *table, *stack, *n_free;
  const int32_t *old_lens, *new_lens;
  int B, M, P, shift;
  int* err;
};

struct Counts {
  int released, wanted;
};
__device__ __forceinline__ Counts add(Counts a, Counts b) {
  return Counts{a.released + b.released, a.wanted + b.wanted};
}

// Exclusive sums over the block's threads; `total` the block's.
__device__ __forceinline__ Counts scan(Counts v, Counts* warp_sum, Counts& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Counts s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const Counts t{__shfl_up_sync(0xffffffffu, s.released, o), __shfl_up_sync(0xffffffffu, s.wanted, o)};
    if (lane >= o) s = add(s, t);
  }
  __syncthreads();
  if (lane == 31) warp_sum[warp] = s;
  __syncthreads();
  Counts before{0, 0};
  total = Counts{0, 0};
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before = add(before, warp_sum[w]);
    total = add(total, warp_sum[w]);
  }
  return Counts{before.released + s.released - v.released, before.wanted + s.wanted - v.wanted};
}

// One cluster.  Each block forms all the sums (entries are few next to their pages); the pages are shared out: a
// team of warps an entry.
__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kThreads) resize_kernel(
    const __grid_constant__ Resize p) {
  namespace cg = cooperative_groups;
  __shared__ Counts warp_sum[kWarps], off[kThreads];
  __shared__ int2 span[kThreads];  // pages an entry had, has
  __shared__ int bad;
  pdl_wait();
  pdl_trigger();
  const cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = (int)cluster.block_rank() * kWarps + (tid >> 5);
  if (tid == 0) bad = 0;
  __syncthreads();
  const int n = *p.n_free;
  const int64_t most = (int64_t)p.M << p.shift;
  // pass 0 counts and checks, 1 releases, 2 takes
  int64_t released = 0, wanted = 0;  // over all entries
  for (int pass = 0; pass < 3; ++pass) {
    Counts done{0, 0};
    for (int b0 = 0; b0 < p.B; b0 += kThreads) {
      const int b = b0 + tid;
      int2 s = make_int2(0, 0);
      bool wrong = false;
      if (b < p.B) {
        const int from = p.old_lens[b], to = p.new_lens[b];
        if (from < 0 || to < 0 || from > most || to > most) wrong = true;
        else s = make_int2((int)(((int64_t)from + (1 << p.shift) - 1) >> p.shift),
                           (int)(((int64_t)to + (1 << p.shift) - 1) >> p.shift));
      }
      if (wrong) bad = 1;
      Counts total;
      const Counts at = add(done, scan(Counts{max(s.x - s.y, 0), max(s.y - s.x, 0)}, warp_sum, total));
      span[tid] = s;
      off[tid] = at;
      done = add(done, total);
      if (pass == 0) released += total.released, wanted += total.wanted;
      __syncthreads();
      // Each entry's pages by a team of warps.  Pass 0: all blocks check all of them, so that all decide alike.
      const int entries = min(kThreads, p.B - b0);
      const int warps = pass == 0 ? kWarps : kWarps * kCluster, mine = pass == 0 ? tid >> 5 : warp;
      const int team = max(1, warps / entries), lanes = team * 32;
      for (int e = mine / team; e < entries && mine / team < warps / team; e += warps / team) {
        const int2 w = span[e];
        const Counts o = off[e];
        int32_t* row = p.table + (int64_t)(b0 + e) * p.M;
        const int i0 = mine % team * 32 + lane;
        if (pass == 0) {
          for (int j = w.y + i0; j < w.x; j += lanes)
            if ((unsigned)row[j] >= (unsigned)p.P) bad = 1;
        } else if (pass == 1) {
          for (int j = w.y + i0; j < w.x; j += lanes) {
            p.stack[n + (int)released - 1 - (o.released + j - w.y)] = row[j];
            row[j] = -1;
          }
        } else {
          for (int j = w.x + i0; j < w.y; j += lanes) {
            int32_t* top = p.stack + n + (int)released - 1 - (o.wanted + j - w.x);
            row[j] = *top;
            *top = -1;
          }
        }
      }
      __syncthreads();
    }
    if (pass == 0) {
      if (n < 0 || n > p.P || n + released > p.P || wanted > n + released) {
        if (tid == 0) bad = 1;
      } else {  // the pages that were on the stack before and are taken now
        for (int i = tid; i < (int)(wanted - released); i += kThreads)
          if ((unsigned)p.stack[n - 1 - i] >= (unsigned)p.P) bad = 1;
      }
      __syncthreads();
      if (bad) {  // the same in every block
        if (tid == 0) record_error(p.err, HCLSM_ERR_SHAPE);
        return;
      }
    }
    cluster.sync();  // the checks before the first change, the releases before the first taking
  }
  if (warp == 0 && lane == 0) *p.n_free = n + (int)(released - wanted);
}

struct Slots {
  const int32_t *table, *start, *count;
  int32_t* slots;
  int B, M, n, shift;
};

__global__ void __launch_bounds__(256) slots_kernel(const __grid_constant__ Slots p) {
  pdl_wait();
  pdl_trigger();
  const int64_t total = (int64_t)p.B * p.n;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int b = (int)(i / p.n), j = (int)(i - (int64_t)b * p.n);
    const int64_t at = (int64_t)p.start[b] + j;
    int slot = -1;
    if (at >= 0 && at < ((int64_t)p.M << p.shift) && (!p.count || j < p.count[b])) {
      const int page = p.table[(int64_t)b * p.M + (at >> p.shift)];
      if (page >= 0) slot = (int)((uint32_t)page << p.shift | ((uint32_t)at & ((1u << p.shift) - 1)));
    }
    p.slots[i] = slot;
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

extern "C" int hclsm_pages_resize(int32_t* table, int32_t B, int32_t M, int32_t* stack, int32_t* n_free, int32_t P,
                                  int32_t page, const int32_t* old_lens, const int32_t* new_lens, void* stream) {
  if (B < 0 || M < 0 || P < 0 || !pages::power_of_2(page)) return HCLSM_ERR_SHAPE;
  if ((int64_t)P * page > 0x7fffffff) return HCLSM_ERR_SHAPE;
  if (B == 0) return HCLSM_OK;
  if ((!table && M) || (!stack && P) || !n_free || !old_lens || !new_lens) return HCLSM_ERR_NULL;
  pages::Resize p = {table, stack, n_free, old_lens, new_lens, B, M, P, pages::log2_of(page), device_err_ptr()};
  return launch_pdl(pages::resize_kernel, pages::kCluster, pages::kThreads, 0, static_cast<cudaStream_t>(stream), p);
}

extern "C" int hclsm_page_slots(const int32_t* table, int32_t B, int32_t M, int32_t page, const int32_t* start,
                                const int32_t* count, int32_t n, int32_t* slots, void* stream) {
  if (B < 0 || M < 0 || n < 0 || !pages::power_of_2(page)) return HCLSM_ERR_SHAPE;
  const int64_t total = (int64_t)B * n;
  if (total == 0) return HCLSM_OK;
  if ((!table && M) || !start || !slots) return HCLSM_ERR_NULL;
  pages::Slots p = {table, start, count, slots, B, M, n, pages::log2_of(page)};
  const int64_t blocks = (total + 255) / 256, most = (int64_t)num_sms() * 32;
  return launch_pdl(pages::slots_kernel, (unsigned)(blocks < most ? blocks : most), 256, 0,
                    static_cast<cudaStream_t>(stream), p);
}
