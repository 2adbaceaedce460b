// Passes of the decaying linear attention in bf16 on the 5th-generation tensor cores (decay.cuh has the mathematics).
//
// A block takes one segment of one head, chunk after chunk of 128 tokens:
//   A = x k^T                 128 x 128, fp32 in TMEM
//   P = A w g^|i-j| as bf16 over A (the A operand of the next product), zero outside the pass's past
//   y = f (P v + g^{i+1-r} x T)   two accumulators, joined by the thread of the row
//   T = g^m T + (w k)^T v     the product in TMEM, T in registers in fp32, w_j = w g^{m-1-j+r}
// The state is returned in fp32, so w k is not rounded to bf16: it enters as NP = 3 bf16 pieces (2 where the state is
// only read by later chunks), smallest first.  The tensor cores cut fp32 sums off instead of rounding them, always
// towards zero: so only a chunk's sum is theirs, and chunks are added in registers.  For x T the state is rounded
// to bf16 once, as P is.
// Warps: TMA, MMA, warpgroups of the state (weighted pieces of k, T) and warpgroups of the rows (P, y).
// A chunk moves 4 tiles and forms 6 products of a tile's size (5 with two pieces), so memory would be the bound; what is: a
// chunk's chain of products, weights and products, two blocks an SM with heads of 64 (issue 50 %, L1 38 + 38 % for the
// threads' and the tensor cores' shares), one with 128 (44 %, 35 + 36 %).  256 heads of 64, 8192 tokens: 229 us,
// 4.7 TB/s; 128 heads of 128: 210 us, 5.1 TB/s, and 259 where the state is returned.  All loops are kept short:
// unrolled ones missed the instruction cache (a chunk of heads of 64 from 15000 cycles to 7000, two blocks an SM).
#include "decay.cuh"
#include "xattn_tc.cuh"

namespace hclsm {
namespace decay {

using namespace ::hclsm::tc;
using xattn::kRowBytes;
using xattn::make_map;
using xattn::mappable;
using xattn::pack_bf16;

struct Maps {
  CUtensorMap x[kMost], k[kMost], v[kMost], y[kMost];
};

constexpr int kTok = 128;                     // tokens of a chunk
constexpr int kBlock = kTok * (int)kRowBytes; // 64 dims of a staged tile

// SMALL: heads of 64 with two blocks an SM; without it, where blocks are no more than SMs, a second warpgroup for the
// rows and TMEM of its own for x T make a chunk's chain shorter (48 heads of 2048 tokens, forward: 46 -> 36 us; 160 heads of
// 1024 tokens, more blocks than SMs: 31 us with two an SM, 41 with one).
template <int DX, int DY, int NP, bool SMALL> struct Shape {
  static constexpr bool kSmall = SMALL;
  static constexpr int kWgT = 2, kWg = kSmall ? 1 : 2;  // warpgroups of the state, of the rows: they share out the columns
  static constexpr int kX = DX / 64 * kBlock, kV = DY / 64 * kBlock;
  static constexpr int kT = DY / 64 * DX * (int)kRowBytes;  // bf16 copy of the state
  // y goes out by way of shared memory: a thread's own row is a line for each store, and those took a quarter of the L1's
  // cycles.  With three pieces there is no room beside v: with 128 dims y goes over it and the next v waits until y has left
  // (4 chunks of one head 22.6 -> 20.0 us); with 64, where the wait cost more (128 heads of 2048 tokens 50.7 -> 56.9 us), y
  // is stored by rows.
  static constexpr bool kStaged = DY / kWg == 64 && (NP == 2 || !kSmall), kOverV = NP == 3 && DX == 128 && DY == 128;
  static constexpr int kY = kStaged && !kOverV ? kV : 0;
  static constexpr size_t kBytes = 2 * kX + kV + NP * kX + kT + kY + 1024;
  static constexpr int kThreads = (kWgT + kWg) * 128 + 64;
  // columns of A and P (0), y, x T (small: y's sum starts from it), the state's products
  static constexpr uint32_t kColY = 128, kColXt = kSmall ? kColY : 256, kColT = kSmall ? 192 : 384;
  static constexpr uint32_t kCols = kSmall ? 256 : 512;
  static constexpr int kPerSm = kSmall ? 2 : 1;
};

// 16-byte piece c of row r of a tile of ROWS rows: 64 dims (8 pieces) a block, 128-byte swizzle.  32-bit addresses that are
// formed where they are used: as pointers, kept over the loop, they cost the state's threads their registers.
template <int ROWS> struct RowAt {
  uint32_t base, turn;
  __device__ __forceinline__ RowAt(uint32_t tile, int r) : base(tile + (uint32_t)r * kRowBytes), turn((uint32_t)(r & 7) << 4) {
    asm volatile("" : "+r"(base), "+r"(turn));
  }
  __device__ __forceinline__ uint32_t operator()(int c) const {
    return base + (uint32_t)(c >> 3) * (ROWS * kRowBytes) + (((uint32_t)(c & 7) << 4) ^ turn);
  }
};
__device__ __forceinline__ uint4 ld_shared(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ void st_shared(uint32_t at, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ void store32(__nv_bfloat16* p, const uint32_t (&w)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
               "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

// 8 columns of this warp's lanes: the state's threads have no registers for more beside T.
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, float (&v)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
               : "r"(taddr));
  tmem_wait_ld();
  tmem_pin<8>(v);
}

// NP bf16 pieces of w times a row's dims [8 c0, 8 (c0 + N)), to the same place of the tile at `to` and NP - 1 tiles of
// `step` bytes behind.
template <int NP, int N>
__device__ __forceinline__ void weigh_row(uint32_t from, uint32_t to, int step, int row, int c0, float w) {
  const RowAt<kTok> at(from, row);
  uint4 raw[N];
#pragma unroll
  for (int c = 0; c < N; ++c) raw[c] = ld_shared(at(c0 + c));
#pragma unroll
  for (int c = 0; c < N; ++c) {
    const uint32_t in[4] = {raw[c].x, raw[c].y, raw[c].z, raw[c].w};
    uint32_t q[NP][4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float2 v = mul2(make_float2(__uint_as_float(in[e] << 16), __uint_as_float(in[e] & 0xffff0000u)), make_float2(w, w));
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const uint32_t t = q[i][e] = pack_bf16(v.x, v.y);
        if (i + 1 < NP)
          v = fma2(make_float2(__uint_as_float(t << 16), __uint_as_float(t & 0xffff0000u)), make_float2(-1.0f, -1.0f), v);
      }
    }
    const uint32_t dst = at(c0 + c) + (to - from);
#pragma unroll
    for (int i = 0; i < NP; ++i) st_shared(dst + i * step, q[i][0], q[i][1], q[i][2], q[i][3]);
  }
}
// Zeros for a row behind the length, which is no operand whatever it holds: dims [8 c0, 8 c1) of the n tiles from `to`, `step`
// bytes apart.
__device__ __forceinline__ void clear_row(uint32_t to, int step, int n, int row, int c0, int c1) {
#pragma unroll 1
  for (int i = 0; i < n; ++i)
#pragma unroll 1
    for (int c = c0; c < c1; ++c) st_shared(RowAt<kTok>(to + i * step, row)(c), 0, 0, 0, 0);
}

template <int DX, int DY, int NP, bool SMALL>
__global__ void __launch_bounds__(Shape<DX, DY, NP, SMALL>::kThreads, Shape<DX, DY, NP, SMALL>::kPerSm)
    tc_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Batch bt) {
  const int which = (int)(blockIdx.x % bt.n);
  const Pass& p = bt.p[which];
  using Sh = Shape<DX, DY, NP, SMALL>;
  constexpr int WGT = Sh::kWgT, WG = Sh::kWg;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  // with 64 dims the update's products read 64 rows behind a piece of k, for rows of the result that nobody reads: the
  // pieces come first
  unsigned char *sP = smem, *sX = sP + NP * Sh::kX, *sK = sX + Sh::kX, *sV = sK + Sh::kX, *sY = sV + (Sh::kOverV ? 0 : Sh::kV),
                *sT = sV + Sh::kV + Sh::kY;
  __shared__ uint32_t s_tmem;
  __shared__ volatile int s_abort;
  __shared__ __align__(16) float s_pow[32];  // w g^(distance of a block's j to its end on the later side)
  __shared__ float2 s_g[2];  // decays of a whole chunk and of the incomplete one
  constexpr int kBars = 13;
  __shared__ uint64_t bars[kBars];
  uint64_t *x_full = bars, *k_full = bars + 1, *v_full = bars + 2, *s_full = bars + 3, *p_ready = bars + 4,
           *t_ready = bars + 5, *y_done = bars + 6, *y_free = bars + 7, *x_free = bars + 8, *t_done = bars + 9,
           *w_ready = bars + 10, *y_left = bars + 11, *drain = bars + 12;
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  constexpr int kTmaWarp = (WGT + WG) * 4, kMmaWarp = kTmaWarp + 1;
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)),
                 "r"(Sh::kCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (tid == 0) {
    s_abort = 0;
    for (uint64_t* b = bars; b < bars + kBars; ++b)
      mbar_init(b, b == t_ready || b == w_ready ? WGT * 128 : b == p_ready || b == y_free ? WG * 128 : b == y_left ? WG * 4 : 1);
    fence_mbar_init();
  }
  pdl_wait();
  pdl_trigger();
  const uint32_t block = blockIdx.x / bt.n;
  const int seg = (int)(block % p.segs);
  const int64_t bh = block / p.segs, b = bh / p.H;
  const int h = (int)(bh - b * p.H), r = p.rev ? 1 : 0;
  const int n = length(p, b);
  const float l2 = log2_decay(p.log_decay, h);
  if (tid < 32) s_pow[tid] = p.w * ex2(l2 * (float)(r ? tid : 31 - tid));
  if (warp == kTmaWarp && lane < 2) s_g[lane] = chunk_decay(p.log_decay, h, lane ? n % kTok : kTok);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  const int c_lo = seg * p.seg_chunks, c_end = min(c_lo + p.seg_chunks, chunks_of(p.L, kTok));
  const int chunks = max(min(c_end, chunks_of(n, kTok)) - c_lo, 0);  // with valid tokens
  auto wait = [&](uint64_t* bar, uint32_t parity) { return mbar_wait_or(bar, parity & 1, &s_abort, p.err); };
  // the whole warp goes on or gives up together
  auto wait_all = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)) != 0; };
  auto first_token = [&](int it) { return (p.rev ? c_lo + chunks - 1 - it : c_lo + it) * kTok; };
  const bool state_out = p.segs == 1 && p.last;
  const int64_t sz = (int64_t)p.Dk * p.Dv;

  int asked_x = 0, asked_k = 0, asked_v = 0;  // copies (lane 0 of the TMA warp)
  if (warp == kTmaWarp) {
    if (lane == 0) {
      for (int it = 0; it < chunks; ++it) {
        const int t0 = first_token(it);
        // in the order in which the chunk before gives them up
        if (it > 0 && (!wait(s_full, it - 1) || !wait(w_ready, it - 1))) break;
        mbar_expect_tx(k_full, Sh::kX);
        for (int d = 0; d < DX / 64; ++d) tma_load_4d(sK + d * kBlock, &maps.k[which], d * 64, t0, h, (int)b, k_full);
        asked_k = it + 1;
        if (it > 0 && !wait(x_free, it - 1)) break;
        mbar_expect_tx(x_full, Sh::kX);
        for (int d = 0; d < DX / 64; ++d) tma_load_4d(sX + d * kBlock, &maps.x[which], d * 64, t0, h, (int)b, x_full);
        asked_x = it + 1;
        if (it > 0 && !wait(Sh::kOverV ? y_left : y_done, it - 1)) break;  // behind the state's update as well
        mbar_expect_tx(v_full, Sh::kV);
        for (int d = 0; d < DY / 64; ++d) tma_load_4d(sV + d * kBlock, &maps.v[which], d * 64, t0, h, (int)b, v_full);
        asked_v = it + 1;
      }
    }
  } else if (warp == kMmaWarp) {
    const uint32_t one = elect_one();
    const int ny = (p.Dv + 15) / 16 * 16, kx = (p.Dk + 15) / 16;
    const uint32_t id_s = idesc_bf16(kTok, kTok, false, false), id_y = idesc_bf16(kTok, ny, false, true),
                   id_t = idesc_bf16(128, ny, true, true);
    const uint64_t d_x = smem_desc_sw128(smem_u32(sX), 16, 1024), d_k = smem_desc_sw128(smem_u32(sK), 16, 1024),
                   d_v = smem_desc_sw128(smem_u32(sV), kBlock, 1024),
                   d_t = smem_desc_sw128(smem_u32(sT), DX * kRowBytes, 1024),
                   d_p = smem_desc_sw128(smem_u32(sP), kBlock, 1024);
    for (int it = 0; it < chunks; ++it) {
      if (!wait_all(k_full, it) || !wait_all(x_full, it)) break;
      // over the chunk before's weights: products run in order
      tc_fence_after();
#pragma unroll
      for (int k = 0; k < DX / 16; ++k) {
        const uint32_t off = (k >> 2) * kBlock + (k & 3) * 32;
        if (k < kx) umma_ss(one, tmem, desc_at(d_x, off), desc_at(d_k, off), id_s, k != 0);
      }
      umma_done(one, s_full);
      // y_free: the row's threads have read the chunk before's
      if (!wait_all(t_ready, it) || (it > 0 && !wait_all(y_free, it - 1))) break;
      tc_fence_after();
#pragma unroll
      for (int k = 0; k < DX / 16; ++k)
        if (k < kx)
          umma_ss(one, tmem + Sh::kColXt, desc_at(d_x, (k >> 2) * kBlock + (k & 3) * 32),
                  desc_at(d_t, k * 16 * kRowBytes), id_y, k != 0);
      umma_done(one, x_free);
      if (!wait_all(w_ready, it) || !wait_all(v_full, it)) break;
      tc_fence_after();
#pragma unroll
      for (int i = NP - 1; i >= 0; --i)
#pragma unroll
        for (int k = 0; k < kTok / 16; ++k)
          umma_ss(one, tmem + Sh::kColT, desc_at(d_p, i * Sh::kX + k * 16 * kRowBytes), desc_at(d_v, k * 16 * kRowBytes),
                  id_t, !(i == NP - 1 && k == 0));
      umma_done(one, t_done);
      if (!wait_all(p_ready, it)) break;
      tc_fence_after();
#pragma unroll
      for (int k = 0; k < kTok / 16; ++k)
        umma_ts(one, tmem + Sh::kColY, tmem + k * 8 + (WG == 2 && k >= 4 ? 32 : 0), desc_at(d_v, k * 16 * kRowBytes), id_y,
                Sh::kSmall || k != 0);
      umma_done(one, y_done);
    }
  } else if (warp < WGT * 4) {
    // ---- the state --------------------------------------------------------------------------
    const int row = tid & 127, half = tid >> 7;  // token, or row of T; columns of this warpgroup
    constexpr int kCols = DY / WGT, kDims = DX / WGT;
    const int y0 = half * kCols;
    const bool holds = (warp & 3) * 32 < DX;  // this warp's lanes are rows of T
    const uint32_t tT = tmem + ((uint32_t)((warp & 3) * 32) << 16) + Sh::kColT + y0;
    const float2 whole = s_g[0], cut_off = s_g[1];
    float2 T[kCols / 2];
#pragma unroll
    for (int e = 0; e < kCols / 2; ++e) T[e] = make_float2(0.0f, 0.0f);
    if (holds) {  // the first state as if a chunk's sum
      const float* from = p.segs > 1 ? p.part + (bh * p.segs + seg) * sz : p.init ? p.init + bh * sz : nullptr;
      const bool turned = p.segs == 1 && p.init_t;
      const int64_t at = turned ? row + (int64_t)y0 * p.Dk : (int64_t)row * p.Dv + y0, step = turned ? p.Dk : 1;
#pragma unroll 1
      for (int c = 0; c < kCols; c += 16) {
        uint32_t w[16];
#pragma unroll
        for (int e = 0; e < 16; ++e)
          w[e] = from && row < p.Dk && y0 + c + e < p.Dv ? __float_as_uint(from[at + (c + e) * step]) : 0u;
        tmem_st16(tT + c, w);
      }
      tmem_wait_st();
    }
    // T behind m more tokens, whose products are complete
    auto advance = [&](int m) {
      tc_fence_after();
      const float2 g = m == kTok ? whole : cut_off;
      if (!holds) return;
#pragma unroll
      for (int c = 0; c < kCols; c += 8) {
        float v[8];
        tmem_ld8(tT + c, v);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float2& t = T[c / 2 + e];
          t = fma2(t, make_float2(g.x, g.x), fma2(t, make_float2(g.y, g.y), make_float2(v[2 * e], v[2 * e + 1])));
        }
      }
    };
    bool ok = true;
    int m = kTok;  // tokens of the chunk before (the first state: T is zero)
    for (int it = 0; it < chunks && ok; ++it) {
      if (it > 0 && !(ok = wait_all(t_done, it - 1))) break;
      advance(m);
      m = min(n - first_token(it), kTok);
      // T in bf16, for x T
      if (it > 0 && !(ok = wait_all(x_free, it - 1))) break;  // the copy before has been read
      if (holds) {
        const RowAt<DX> at(smem_u32(sT), row);
#pragma unroll
        for (int c = 0; c < kCols; c += 8) {
          uint32_t q[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) q[e] = pack_bf16(T[c / 2 + e].x, T[c / 2 + e].y);
          st_shared(at(y0 / 8 + c / 8), q[0], q[1], q[2], q[3]);
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      tc_fence_before();
      mbar_arrive(t_ready);
      // the pieces of w k
      if (!(ok = wait_all(k_full, it))) break;
      const int c0 = half * (kDims / 8);
      const float w = p.w * ex2(l2 * (float)(p.rev ? row + 1 : m - 1 - row));
#pragma unroll 1
      for (int c = 0; c < kDims / 8; c += 2) weigh_row<NP, 2>(smem_u32(sK), smem_u32(sP), Sh::kX, row, c0 + c, w);
      if (m < kTok) {
        if (!(ok = wait_all(v_full, it))) break;
        if (row >= m) {
          clear_row(smem_u32(sP), Sh::kX, NP, row, c0, c0 + kDims / 8);
          clear_row(smem_u32(sV), 0, 1, row, y0 / 8, (y0 + kCols) / 8);
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      tc_fence_before();  // the products' sum has been read
      mbar_arrive(w_ready);
    }
    if (ok && chunks > 0) {
      ok = wait_all(t_done, chunks - 1);
      if (state_out && ok) advance(m);
    } else if (state_out && ok) {
      advance(kTok);  // no token: the first state alone
    }
    if (state_out && ok && row < p.Dk) {
      float* to = p.last + bh * sz + (int64_t)row * p.Dv + y0;
#pragma unroll
      for (int e = 0; e < kCols; e += 4)
        if (y0 + e < p.Dv)
          *reinterpret_cast<float4*>(to + e) =
              make_float4(T[e / 2].x, T[e / 2].y, T[e / 2 + 1].x, T[e / 2 + 1].y);
    }
  } else {
    // ---- the rows ---------------------------------------------------------------------------
    const int row = tid & 127, half = (tid >> 7) - WGT;  // token; columns of this warpgroup
    const uint32_t tS = tmem + ((uint32_t)((warp & 3) * 32) << 16), tY = tS + Sh::kColY, tX = tS + Sh::kColXt;
    constexpr int kCols = DY / WG, kBlocks = 4 / WG;
    const int y0 = half * kCols, i0 = (warp & 3) * 32;
    const bool wide = p.Dv % 16 == 0 && reinterpret_cast<uintptr_t>(p.y) % 32 == 0;  // rows of whole 32 bytes
    // the log2 of a decay above which g^-31 stays below 2^125 and w g^31 above 2^-125
    const float near = fminf(-4.0f - fminf(__log2f(p.w), 0.0f) * (1.0f / 31.0f), 0.0f);
    bool ok = true;
    for (int it = 0; it < chunks && ok; ++it) {
      const int t0 = first_token(it), m = min(n - t0, kTok);
      const int place = p.rev ? m - 1 - row : row;
      if (!(ok = wait_all(s_full, it))) break;
      tc_fence_after();
#pragma unroll 1
      for (int q = 0; q < kBlocks; ++q) {
        const int j0 = (half * kBlocks + q) * 32;
        const bool past = p.rev ? j0 > i0 : j0 < i0, now = j0 == i0;  // the same for the whole warp
        uint32_t pw[16];
        if ((past || now) && j0 < m) {
          float v[32];
          tmem_ld32_nowait(tS + j0, v);
          // the columns [first, last] count
          const int first = p.rev ? max(row - j0, 0) : 0, last = min(p.rev ? 31 : min(row - j0, 31), m - 1 - j0);
          const uint32_t on = first <= last && first < 32 ? (0xffffffffu >> (31 - (last - first))) << first : 0u;
          if (past || l2 > near) {
            // g^|i-j| as the power of i's distance to the block's end on the later side times that of j's; on the
            // diagonal the first is up to g^-31 and the second, with w, down to w g^31, which fp32 holds above `near`: so the
            // score comes last
            const float a = ex2(l2 * (float)(p.rev ? j0 - row : row - j0 - 31));
            tmem_wait_ld();
            tmem_pin<32>(v);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float4 t = *reinterpret_cast<const float4*>(s_pow + e * 4);
              float2 lo = mul2(make_float2(t.x, t.y), make_float2(a, a)), hi = mul2(make_float2(t.z, t.w), make_float2(a, a));
              lo = mul2(lo, make_float2(v[4 * e], v[4 * e + 1]));
              hi = mul2(hi, make_float2(v[4 * e + 2], v[4 * e + 3]));
              v[4 * e] = lo.x, v[4 * e + 1] = lo.y, v[4 * e + 2] = hi.x, v[4 * e + 3] = hi.y;
            }
          } else {
            const float step = p.rev ? l2 : -l2, base = (p.rev ? -l2 : l2) * (float)(row - j0);
            tmem_wait_ld();
            tmem_pin<32>(v);
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] *= p.w * ex2(fmaf(step, (float)e, base));
          }
          if (!past || j0 + 32 > m) {  // select, not multiply: a later token's score may be NaN, its power inf
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] = on >> e & 1u ? v[e] : 0.0f;
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) pw[e] = pack_bf16(v[2 * e], v[2 * e + 1]);
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) pw[e] = 0;
        }
        // over scores that this thread has read
        tmem_st16(tS + half * 64 + q * 16, pw);
      }
      const float lead = ex2(l2 * (float)(place + 1 - r));
      if constexpr (Sh::kSmall) {  // x T times g^{i+1-r}: what P v is added to
        if (!(ok = wait_all(x_free, it))) break;
        tc_fence_after();
#pragma unroll 1
        for (int c = 0; c < kCols; c += 16) {
          float a[16];
          tmem_ld16_nowait(tY + y0 + c, a);
          tmem_wait_ld();
          tmem_pin<16>(a);
          uint32_t q[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) q[e] = __float_as_uint(a[e] * lead);
          tmem_st16(tY + y0 + c, q);
        }
      }
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(p_ready);
      __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.y) + ((b * p.L + t0 + row) * p.H + h) * (int64_t)p.Dv + y0;
      if (!(ok = wait_all(y_done, it))) break;
      tc_fence_after();
      if (Sh::kStaged && !Sh::kOverV && it > 0) {
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");  // the rows before have left
        __syncwarp();
      }
#pragma unroll 1
      for (int c = 0; c < kCols; c += 16) {
        float a[16], x[16];
        tmem_ld16_nowait(tY + y0 + c, a);
        if constexpr (!Sh::kSmall) tmem_ld16_nowait(tX + y0 + c, x);
        tmem_wait_ld();
        tmem_pin<16>(a);
        if constexpr (!Sh::kSmall) tmem_pin<16>(x);
        if (c + 16 == kCols) {
          tc_fence_before();
          mbar_arrive(y_free);
        }
        uint32_t q[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float2 t = make_float2(a[2 * e], a[2 * e + 1]);
          if constexpr (!Sh::kSmall) t = fma2(make_float2(x[2 * e], x[2 * e + 1]), make_float2(lead, lead), t);
          t = mul2(t, make_float2(p.f, p.f));
          q[e] = pack_bf16(t.x, t.y);
        }
        if constexpr (Sh::kStaged) {
          const RowAt<kTok> at(smem_u32(sY), row);
          const uint32_t keep = row < m ? 0xffffffffu : 0u;  // zeros behind the length
          st_shared(at((y0 + c) / 8), q[0] & keep, q[1] & keep, q[2] & keep, q[3] & keep);
          st_shared(at((y0 + c) / 8 + 1), q[4] & keep, q[5] & keep, q[6] & keep, q[7] & keep);
        } else if (row < m && y0 + c < p.Dv) {
          if (wide) {
            store32(out + c, q);
          } else {
            *reinterpret_cast<uint4*>(out + c) = make_uint4(q[0], q[1], q[2], q[3]);
            if (y0 + c + 8 < p.Dv) *reinterpret_cast<uint4*>(out + c + 8) = make_uint4(q[4], q[5], q[6], q[7]);
          }
        }
      }
      if constexpr (Sh::kStaged) {  // a warp's 32 rows of 64 dims
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0 && t0 + i0 < p.L) {
          asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%1, %2, %3, %4}], [%5];" ::"l"(
                           &maps.y[which]),
                       "r"(y0), "r"(t0 + i0), "r"(h), "r"((int)b), "r"(smem_u32(sY + y0 / 64 * kBlock + i0 * (int)kRowBytes))
                       : "memory");
          asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
        if (Sh::kOverV && lane == 0) {
          asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
          mbar_arrive(y_left);
        }
      }
    }
    if (Sh::kStaged && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    // zeros behind the length
    const int e8 = p.Dv / 8, me = tid - WGT * 128;
    for (int64_t t = max(c_lo * kTok, n) + (int64_t)(me >> 3), end = min((int64_t)c_end * kTok, (int64_t)p.L); t < end;
         t += WG * 16)
      for (int e = me & 7; e < e8; e += 8)
        *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.y) + ((b * p.L + t) * p.H + h) * (int64_t)p.Dv + e * 8) =
            make_uint4(0, 0, 0, 0);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (s_abort) {  // the same for all: nothing writes it after the barrier
    if (warp == kMmaWarp) drain_umma(drain);
    if (warp == kTmaWarp && lane == 0) {
      drain_copies(x_full, asked_x, 1);
      drain_copies(k_full, asked_k, 1);
      drain_copies(v_full, asked_v, 1);
    }
    __syncthreads();
  }
  if (warp == kMmaWarp)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(Sh::kCols) : "memory");
}

// ---- the segments' own sums --------------------------------------------------------------------
// No x and no y: T = sum over the segment of (w_j k_j)^T v_j, w_j to the segment's end, so T is never scaled.  k is free
// when its pieces are written, v has two stages; one chunk's sum is added to the registers while the next one's
// products run.
template <int DX, int DY> struct SumShape {
  static constexpr int kNP = 3, kStages = 2;
  static constexpr int kWg = 2;
  static constexpr int kX = DX / 64 * kBlock, kV = DY / 64 * kBlock;
  static constexpr size_t kBytes = kX + kStages * (size_t)kV + (size_t)kNP * kX + 1024;
  static constexpr int kThreads = kWg * 128 + 64;
  static constexpr uint32_t kCols = 2 * DY;
  static constexpr int kPerSm = DX == 64 && DY == 64 ? 2 : 1;
};

template <int DX, int DY>
__global__ void __launch_bounds__(SumShape<DX, DY>::kThreads, SumShape<DX, DY>::kPerSm)
    sums_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Batch bt) {
  const int which = (int)(blockIdx.x % bt.n);
  const Pass& p = bt.p[which];
  using Sh = SumShape<DX, DY>;
  constexpr int NP = Sh::kNP, ST = Sh::kStages, WG = Sh::kWg;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char *sP = smem, *sK = sP + NP * Sh::kX, *sV = sK + Sh::kX;  // the pieces first, as above
  __shared__ uint32_t s_tmem;
  __shared__ volatile int s_abort;
  constexpr int kBars = 2 * ST + 3;
  __shared__ uint64_t bars[kBars];
  // done: one a stage of v.  The copies wait for products of two chunks ago, and behind one barrier of both stages the
  // products of the chunk between might have ended as well: a wait for the phase before the last does not return.
  uint64_t *full = bars, *done = bars + ST, *k_full = bars + 2 * ST, *ready = k_full + 1, *drain = ready + 1;
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  constexpr int kTmaWarp = WG * 4, kMmaWarp = WG * 4 + 1;
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)),
                 "r"(Sh::kCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (tid == 0) {
    s_abort = 0;
    for (uint64_t* b = bars; b < bars + kBars; ++b) mbar_init(b, b == ready ? WG * 128 : 1);
    fence_mbar_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_wait();
  pdl_trigger();
  const uint32_t tmem = s_tmem;
  const uint32_t block = blockIdx.x / bt.n;
  const int seg = (int)(block % p.segs);
  const int64_t bh = block / p.segs, b = bh / p.H;
  const int h = (int)(bh - b * p.H);
  const int n = length(p, b);
  const float l2 = log2_decay(p.log_decay, h);
  const int lo = seg * p.seg_chunks * kTok;
  const int hi = (int)min((int64_t)lo + p.seg_chunks * kTok, (int64_t)n);  // the segment's end may lie past 31 bits
  const int chunks = hi > lo ? chunks_of(hi - lo, kTok) : 0;
  auto wait = [&](uint64_t* bar, uint32_t parity) { return mbar_wait_or(bar, parity & 1, &s_abort, p.err); };
  auto wait_all = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)) != 0; };
  int asked = 0, asked_k = 0;
  if (warp == kTmaWarp) {
    if (lane == 0)
      for (int it = 0; it < chunks; ++it) {
        const int s = it % ST, t0 = lo + it * kTok;
        if (it > 0 && !wait(ready, it - 1)) break;
        mbar_expect_tx(k_full, Sh::kX);
        for (int d = 0; d < DX / 64; ++d) tma_load_4d(sK + d * kBlock, &maps.k[which], d * 64, t0, h, (int)b, k_full);
        asked_k = it + 1;
        if (it >= ST && !wait(&done[s], it / ST - 1)) break;
        mbar_expect_tx(&full[s], Sh::kV);
        for (int d = 0; d < DY / 64; ++d)
          tma_load_4d(sV + s * Sh::kV + d * kBlock, &maps.v[which], d * 64, t0, h, (int)b, &full[s]);
        asked = it + 1;
      }
  } else if (warp == kMmaWarp) {
    const uint32_t one = elect_one();
    const uint32_t id_t = idesc_bf16(128, (p.Dv + 15) / 16 * 16, true, true);
    const uint64_t d_v = smem_desc_sw128(smem_u32(sV), kBlock, 1024),
                   d_p = smem_desc_sw128(smem_u32(sP), kBlock, 1024);
    for (int it = 0; it < chunks; ++it) {
      if (!wait_all(ready, it) || !wait_all(&full[it % ST], it / ST)) break;
      tc_fence_after();
#pragma unroll
      for (int i = NP - 1; i >= 0; --i)
#pragma unroll
        for (int k = 0; k < kTok / 16; ++k)
          umma_ss(one, tmem + (it & 1) * DY, desc_at(d_p, i * Sh::kX + k * 16 * kRowBytes),
                  desc_at(d_v, it % ST * Sh::kV + k * 16 * kRowBytes), id_t, !(i == NP - 1 && k == 0));
      umma_done(one, &done[it % ST]);
    }
  } else {
    const int row = tid & 127, half = tid >> 7;
    constexpr int kCols = DY / WG, kDims = DX / WG;
    const int y0 = half * kCols;
    const bool holds = (warp & 3) * 32 < DX;
    const uint32_t tT = tmem + ((uint32_t)((warp & 3) * 32) << 16) + y0;
    float T[kCols];
#pragma unroll
    for (int e = 0; e < kCols; ++e) T[e] = 0.0f;
    auto add = [&](int it) {
      if (!holds) return;
#pragma unroll
      for (int c = 0; c < kCols; c += 16) {
        float v[16];
        tmem_ld16_nowait(tT + (it & 1) * DY + c, v);
        tmem_wait_ld();
        tmem_pin<16>(v);
#pragma unroll
        for (int e = 0; e < 16; ++e) T[c + e] += v[e];
      }
    };
    bool ok = true;
    for (int it = 0; it < chunks && ok; ++it) {
      const int s = it % ST, t = lo + it * kTok + row;
      if (!(ok = wait_all(k_full, it))) break;
      // the products that read the pieces are complete
      if (it > 0 && !(ok = wait_all(&done[(it - 1) % ST], (it - 1) / ST))) break;
      const int c0 = half * (kDims / 8);
      const float w = ex2(l2 * (float)(p.rev ? t - lo + 1 : hi - 1 - t));
#pragma unroll 1
      for (int c = 0; c < kDims / 8; c += 4) weigh_row<NP, 4>(smem_u32(sK), smem_u32(sP), Sh::kX, row, c0 + c, w);
      if (hi - lo - it * kTok < kTok) {
        if (!(ok = wait_all(&full[s], it / ST))) break;
        if (t >= hi) {
          clear_row(smem_u32(sP), Sh::kX, NP, row, c0, c0 + kDims / 8);
          clear_row(smem_u32(sV + s * Sh::kV), 0, 1, row, y0 / 8, (y0 + kCols) / 8);
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      tc_fence_before();
      mbar_arrive(ready);
      if (it > 0) {
        tc_fence_after();
        add(it - 1);
      }
    }
    if (ok && chunks > 0 && wait_all(&done[(chunks - 1) % ST], (chunks - 1) / ST)) {
      tc_fence_after();
      add(chunks - 1);
    }
    if (row < p.Dk) {
      float* to = p.part + (bh * p.segs + seg) * ((int64_t)p.Dk * p.Dv) + (int64_t)row * p.Dv + y0;
#pragma unroll
      for (int e = 0; e < kCols; e += 4)
        if (y0 + e < p.Dv)
          *reinterpret_cast<float4*>(to + e) = make_float4(p.w * T[e], p.w * T[e + 1], p.w * T[e + 2], p.w * T[e + 3]);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (s_abort) {
    if (warp == kMmaWarp) drain_umma(drain);
    if (warp == kTmaWarp && lane == 0) {
      drain_copies(k_full, asked_k, 1);
      drain_copies(full, asked, ST);
    }
    __syncthreads();
  }
  if (warp == kMmaWarp)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(Sh::kCols) : "memory");
}

// ---- host ----------------------------------------------------------------------------------
bool tc_ok(const Batch& b) {
  for (int i = 0; i < b.n; ++i) {
    const Pass& p = b.p[i];
    if (!(p.Dk % 8 == 0 && p.Dv % 8 == 0 && mappable(p.x, p.L, p.H, p.B) && mappable(p.k, p.L, p.H, p.B) &&
          mappable(p.v, p.L, p.H, p.B) && reinterpret_cast<uintptr_t>(p.y) % 16 == 0 &&
          reinterpret_cast<uintptr_t>(p.last) % 16 == 0))
      return false;
  }
  return true;
}

void tc_cut(Batch& b) {
  const Pass& p = b.p[0];
  cut(b, kTok, 1.9f, 1.4f, 4.0f, 4.0f, (int64_t)b.n * p.B * p.H, (int64_t)num_sms() * (p.Dk <= 64 && p.Dv <= 64 ? 2 : 1));
}

template <int DX, int DY, int NP, bool SMALL>
int launch(const Batch& b, cudaStream_t st) {
  using Sh = Shape<DX, DY, NP, SMALL>;
  auto fn = tc_kernel<DX, DY, NP, SMALL>;
  // before the maps: encoding one needs the device's context, which this call makes current in a new thread
  if (!set_smem_limit(reinterpret_cast<const void*>(fn), Sh::kBytes)) return HCLSM_ERR_LAUNCH;
  Maps maps;
  for (int i = 0; i < b.n; ++i) {
    const Pass& p = b.p[i];
    if (!make_map(&maps.x[i], p.x, p.Dk, p.L, p.H, p.B, kTok) || !make_map(&maps.k[i], p.k, p.Dk, p.L, p.H, p.B, kTok) ||
        !make_map(&maps.v[i], p.v, p.Dv, p.L, p.H, p.B, kTok))
      return HCLSM_ERR_UNSUPPORTED;
    const View y = xattn::view(hclsm_view{p.y, (int64_t)p.L * p.H * p.Dv, (int64_t)p.H * p.Dv, p.Dv}, p.B, p.L, p.H);
    if (Sh::kStaged && !make_map(&maps.y[i], y, p.Dv, p.L, p.H, p.B, 32)) return HCLSM_ERR_UNSUPPORTED;
  }
  const Pass& p = b.p[0];
  const int64_t grid = (int64_t)b.n * p.B * p.H * p.segs;
  if (grid > 0x7fffffff) return HCLSM_ERR_SHAPE;
  if (p.segs > 1) {
    using Ss = SumShape<DX, DY>;
    auto sums = sums_kernel<DX, DY>;
    if (!set_smem_limit(reinterpret_cast<const void*>(sums), Ss::kBytes)) return HCLSM_ERR_LAUNCH;
    if (const int rc = launch_pdl(sums, (unsigned)grid, Ss::kThreads, Ss::kBytes, st, maps, b)) return rc;
    if (const int rc = join(b, kTok, st)) return rc;
  }
  return launch_pdl(fn, (unsigned)grid, Sh::kThreads, Sh::kBytes, st, maps, b);
}

template <int DX, int DY, bool SMALL>
int launch_np(const Batch& b, cudaStream_t st) {
  bool out = false;  // a state that is returned
  for (int i = 0; i < b.n; ++i) out = out || (b.p[i].last && b.p[i].segs == 1);
  return out ? launch<DX, DY, 3, SMALL>(b, st) : launch<DX, DY, 2, SMALL>(b, st);
}

int tc_run(const Batch& b, cudaStream_t st) {
  const Pass& p = b.p[0];
  if (p.Dk <= 64 && p.Dv <= 64)
    return (int64_t)b.n * p.B * p.H * p.segs <= num_sms() ? launch_np<64, 64, false>(b, st) : launch_np<64, 64, true>(b, st);
  if (p.Dk <= 64) return launch_np<64, 128, false>(b, st);
  return p.Dv <= 64 ? launch_np<128, 64, false>(b, st) : launch_np<128, 128, false>(b, st);
}

}  // namespace decay
}  // namespace hclsm
