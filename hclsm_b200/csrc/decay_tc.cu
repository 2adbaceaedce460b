// Passes of the decaying linear attention in bf16 on the 5th-generation tensor cores (decay.cuh has the mathematics).
//
// A block takes one segment of one head, chunk after chunk of 128 tokens:
//   A = x k^T                 128 x 128, fp32 in TMEM
//   P = A g^|i-j| as bf16 over A (the A operand of the next product), zero outside the pass's past
//   y = f (P v + g^{i+1-r} x T)   two accumulators, joined by the thread of the row
//   T = g^m T + k^T (w v)     fp32 in TMEM, w_j = g^{m-1-j+r}
// The state is returned in fp32, so w v (or w k, whichever is narrower) is not rounded to bf16: it enters as NP = 3
// bf16 pieces (2 where the state is only read by later chunks), each exact product summed in fp32.  For x T the state
// is rounded to bf16 once, as P is.
// Two warps issue: TMA and MMA.  NWG warpgroups do the rest, a thread a row (token, or row of T) and NWG its columns.
#include "decay.cuh"
#include "xattn_tc.cuh"

namespace hclsm {
namespace decay {

using namespace ::hclsm::tc;
using xattn::kRowBytes;
using xattn::make_map;
using xattn::mappable;
using xattn::pack_bf16;

constexpr int kTok = 128;                     // tokens of a chunk
constexpr int kBlock = kTok * (int)kRowBytes; // 64 dims of a staged tile

template <int DX, int DY, int NP> struct Shape {
  static constexpr bool kScaleV = DY <= DX;   // the operand of the state's update that takes the weights
  static constexpr int kNwg = DX == 64 && DY == 64 ? 1 : 2;
  static constexpr int kX = DX / 64 * kBlock, kV = DY / 64 * kBlock;
  static constexpr int kPiece = kScaleV ? kV : kX;
  static constexpr int kT = DY / 64 * DX * (int)kRowBytes;  // bf16 copy of the state
  static constexpr int kBars = 10;
  static constexpr size_t kBytes = 2 * kX + kV + NP * kPiece + kT + 1024;
  static constexpr int kThreads = kNwg * 128 + 64;
  static constexpr uint32_t kColY = 128, kColXt = DY == 64 ? 64 : 256, kColT = DY == 64 ? 192 : 384;
  static constexpr uint32_t kCols = DY == 64 ? 256 : 512;
  static constexpr int kPerSm = DX == 64 && DY == 64 ? 2 : 1;
};

// Bytes of 16-byte piece c of row r of a tile of `rows` rows, 64 dims (8 pieces) a block, 128-byte swizzle.
__device__ __forceinline__ int swizzled(int rows, int r, int c) {
  return ((c >> 3) * rows + r) * (int)kRowBytes + (((c & 7) ^ (r & 7)) << 4);
}
__device__ __forceinline__ void store32(__nv_bfloat16* p, const uint32_t (&w)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
               "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

template <int DX, int DY, int NP>
__global__ void __launch_bounds__(Shape<DX, DY, NP>::kThreads, Shape<DX, DY, NP>::kPerSm)
    tc_kernel(const __grid_constant__ CUtensorMap mx, const __grid_constant__ CUtensorMap mk,
              const __grid_constant__ CUtensorMap mv, const __grid_constant__ Pass p) {
  using Sh = Shape<DX, DY, NP>;
  constexpr int NWG = Sh::kNwg;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char *sX = smem, *sK = sX + Sh::kX, *sV = sK + Sh::kX, *sP = sV + Sh::kV, *sT = sP + NP * Sh::kPiece;
  __shared__ uint32_t s_tmem;
  __shared__ volatile int s_abort;
  __shared__ __align__(16) float s_pow[32];  // g^n
  __shared__ uint64_t bars[Sh::kBars];
  uint64_t *xk_full = bars, *v_full = bars + 1, *s_full = bars + 2, *p_ready = bars + 3, *t_ready = bars + 4,
           *y_done = bars + 5, *x_free = bars + 6, *t_done = bars + 7, *read = bars + 8, *drain = bars + 9;
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  constexpr int kTmaWarp = NWG * 4, kMmaWarp = NWG * 4 + 1;
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)),
                 "r"(Sh::kCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (tid == 0) {
    s_abort = 0;
    for (uint64_t* b = bars; b < bars + Sh::kBars; ++b) mbar_init(b, b == p_ready || b == t_ready || b == read ? NWG * 128 : 1);
    fence_mbar_init();
  }
  pdl_wait();
  pdl_trigger();
  const int seg = (int)(blockIdx.x % p.segs);
  const int64_t bh = blockIdx.x / p.segs, b = bh / p.H;
  const int h = (int)(bh - b * p.H), r = p.rev ? 1 : 0;
  const int n = length(p, b);
  const float l2 = log2_decay(p.log_decay, h);
  if (tid < 32) s_pow[tid] = ex2(l2 * (float)tid);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  const int c_lo = seg * p.seg_chunks, c_end = min(c_lo + p.seg_chunks, (p.L + kTok - 1) / kTok);
  const int chunks = max(min(c_end, (n + kTok - 1) / kTok) - c_lo, 0);  // with valid tokens
  auto wait = [&](uint64_t* bar, uint32_t parity) { return mbar_wait_or(bar, parity & 1, &s_abort, p.err); };
  // the whole warp goes on or gives up together
  auto wait_all = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)) != 0; };
  auto first_token = [&](int it) { return (p.rev ? c_lo + chunks - 1 - it : c_lo + it) * kTok; };
  const bool state_out = p.segs == 1 && p.last;

  int asked_xk = 0, asked_v = 0;  // copies (lane 0 of the TMA warp)
  if (warp == kTmaWarp) {
    if (lane == 0) {
      for (int it = 0; it < chunks; ++it) {
        const int t0 = first_token(it);
        if (it > 0 && !wait(x_free, it - 1)) break;
        mbar_expect_tx(xk_full, 2 * Sh::kX);
        for (int d = 0; d < DX / 64; ++d) tma_load_4d(sX + d * kBlock, &mx, d * 64, t0, h, (int)b, xk_full);
        asked_xk = it + 1;
        // given up between the two: k is asked for all the same, so that the barrier's bytes arrive
        const bool ok = it == 0 || wait(t_done, it - 1);
        if (!ok) mbar_wait(t_done, (it - 1) & 1);
        for (int d = 0; d < DX / 64; ++d) tma_load_4d(sK + d * kBlock, &mk, d * 64, t0, h, (int)b, xk_full);
        if (!ok) break;
        mbar_expect_tx(v_full, Sh::kV);
        for (int d = 0; d < DY / 64; ++d) tma_load_4d(sV + d * kBlock, &mv, d * 64, t0, h, (int)b, v_full);
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
                   d_kt = smem_desc_sw128(smem_u32(sK), kBlock, 1024),
                   d_p = smem_desc_sw128(smem_u32(sP), kBlock, 1024);
    for (int it = 0; it < chunks; ++it) {
      if (!wait_all(xk_full, it)) break;
      tc_fence_after();
      // Over the chunk before's weights (products run in order) and, with 64 value dims, its x T: a row's thread has
      // read that when it arrives on t_ready.
      if (DY == 64 && it > 0 && !wait_all(t_ready, it)) break;
      tc_fence_after();
#pragma unroll
      for (int k = 0; k < DX / 16; ++k) {
        const uint32_t off = (k >> 2) * kBlock + (k & 3) * 32;
        if (k < kx) umma_ss(one, tmem, desc_at(d_x, off), desc_at(d_k, off), id_s, k != 0);
      }
      umma_done(one, s_full);
      if (!wait_all(v_full, it) || !wait_all(t_ready, it) || !wait_all(p_ready, it)) break;
      tc_fence_after();
#pragma unroll
      for (int k = 0; k < DX / 16; ++k)
        if (k < kx)
          umma_ss(one, tmem + Sh::kColXt, desc_at(d_x, (k >> 2) * kBlock + (k & 3) * 32),
                  desc_at(d_t, k * 16 * kRowBytes), id_y, k != 0);
      umma_done(one, x_free);
#pragma unroll
      for (int k = 0; k < kTok / 16; ++k)
        umma_ts(one, tmem + Sh::kColY, tmem + k * 8, desc_at(d_v, k * 16 * kRowBytes), id_y, k != 0);
      umma_done(one, y_done);
#pragma unroll
      for (int i = 0; i < NP; ++i)
#pragma unroll
        for (int k = 0; k < kTok / 16; ++k) {
          const uint64_t pd = desc_at(d_p, i * Sh::kPiece + k * 16 * kRowBytes);
          umma_ss(one, tmem + Sh::kColT, Sh::kScaleV ? desc_at(d_kt, k * 16 * kRowBytes) : pd,
                  Sh::kScaleV ? pd : desc_at(d_v, k * 16 * kRowBytes), id_t, 1);
        }
      umma_done(one, t_done);
    }
  } else {
    const int row = tid & 127, half = tid >> 7;  // token, or row of the state; columns of this warpgroup
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + lanes, tY = tS + Sh::kColY, tX = tS + Sh::kColXt, tT = tS + Sh::kColT;
    constexpr int kYCols = DY / NWG, kPDims = (Sh::kScaleV ? DY : DX) / NWG, kBlocks = 4 / NWG;
    const int y0 = half * kYCols;
    const bool holds_t = (warp & 3) * 32 < DX;  // this warp's lanes are rows of the state
    const float2 whole = chunk_decay(p.log_decay, h, kTok);
    const int64_t sz = (int64_t)p.Dk * p.Dv;
    bool ok = true;
    if (holds_t) {
#pragma unroll 1
      for (int c = 0; c < kYCols; c += 16) {
        uint32_t w[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int col = y0 + c + e;
          float v = 0.0f;
          if (row < p.Dk && col < p.Dv) {
            if (p.segs > 1) v = p.part[(bh * p.segs + seg) * sz + (int64_t)row * p.Dv + col];
            else if (p.init) v = p.init_f * p.init[bh * sz + (p.init_t ? (int64_t)col * p.Dk + row : (int64_t)row * p.Dv + col)];
          }
          w[e] = __float_as_uint(v);
        }
        tmem_st16(tT + y0 + c, w);
      }
      tmem_wait_st();
    }
    for (int it = 0; it < chunks && ok; ++it) {
      const int t0 = first_token(it), m = min(n - t0, kTok);
      const int place = p.rev ? m - 1 - row : row;
      // ---- the state: its bf16 copy, then times the chunk's decay
      if (it > 0) {
        if (!(ok = wait_all(t_done, it - 1))) break;
        tc_fence_after();
      }
      if (holds_t) {
        const float2 g = m == kTok ? whole : chunk_decay(p.log_decay, h, m);
#pragma unroll 1
        for (int c = 0; c < kYCols; c += 16) {
          float v[16];
          tmem_ld16_nowait(tT + y0 + c, v);
          tmem_wait_ld();
          tmem_pin<16>(v);
          uint32_t w[16], q[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) q[e] = pack_bf16(v[2 * e], v[2 * e + 1]);
#pragma unroll
          for (int e = 0; e < 16; ++e) w[e] = __float_as_uint(fmaf(v[e], g.x, v[e] * g.y));
          tmem_st16(tT + y0 + c, w);
          const int at = (y0 + c) / 8;
          *reinterpret_cast<uint4*>(sT + swizzled(DX, row, at)) = make_uint4(q[0], q[1], q[2], q[3]);
          *reinterpret_cast<uint4*>(sT + swizzled(DX, row, at + 1)) = make_uint4(q[4], q[5], q[6], q[7]);
        }
        tmem_wait_st();
      }
      // ---- the weighted operand of the state's update; rows behind the length are no operands
      if (!(ok = wait_all(xk_full, it) && wait_all(v_full, it))) break;
      if (row >= m) {
        for (int c = half; c < DX / 8; c += NWG) *reinterpret_cast<uint4*>(sK + swizzled(kTok, row, c)) = make_uint4(0, 0, 0, 0);
        for (int c = half; c < DY / 8; c += NWG) *reinterpret_cast<uint4*>(sV + swizzled(kTok, row, c)) = make_uint4(0, 0, 0, 0);
      }
      {
        const float w = ex2(l2 * (float)(m - 1 - place + r));
        const unsigned char* from = Sh::kScaleV ? sV : sK;
#pragma unroll 2
        for (int c = half * (kPDims / 8); c < (half + 1) * (kPDims / 8); ++c) {
          const int at = swizzled(kTok, row, c);
          uint32_t q[NP][4] = {};
          if (row < m) {
            const uint4 raw = *reinterpret_cast<const uint4*>(from + at);
            const uint32_t in[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float lo = __uint_as_float(in[e] << 16) * w, hi = __uint_as_float(in[e] & 0xffff0000u) * w;
#pragma unroll
              for (int i = 0; i < NP; ++i) {
                q[i][e] = pack_bf16(lo, hi);
                lo -= __uint_as_float(q[i][e] << 16), hi -= __uint_as_float(q[i][e] & 0xffff0000u);
              }
            }
          }
#pragma unroll
          for (int i = 0; i < NP; ++i)
            *reinterpret_cast<uint4*>(sP + i * Sh::kPiece + at) = make_uint4(q[i][0], q[i][1], q[i][2], q[i][3]);
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      tc_fence_before();
      mbar_arrive(t_ready);
      // ---- P
      if (!(ok = wait_all(s_full, it))) break;
      tc_fence_after();
      uint32_t pw[kBlocks][16];
#pragma unroll
      for (int q = 0; q < kBlocks; ++q) {
        const int j0 = (half * kBlocks + q) * 32, i0 = (warp & 3) * 32;
        const bool past = p.rev ? j0 > i0 : j0 < i0, now = j0 == i0;  // the same for the whole warp
        if (!past && !now) {
#pragma unroll
          for (int e = 0; e < 16; ++e) pw[q][e] = 0;
          continue;
        }
        float v[32];
        tmem_ld32_nowait(tS + j0, v);
        tmem_wait_ld();
        tmem_pin<32>(v);
        if (past && j0 + 32 <= m) {
          // g^|i-j| as the power of i's distance to the block's near end times that of j's
          const float a = ex2(l2 * (float)(p.rev ? j0 - row : row - j0 - 31));
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float4 t = *reinterpret_cast<const float4*>(s_pow + (p.rev ? e : 7 - e) * 4);
            float2 lo = mul2(make_float2(v[4 * e], v[4 * e + 1]), make_float2(a, a)),
                   hi = mul2(make_float2(v[4 * e + 2], v[4 * e + 3]), make_float2(a, a));
            lo = mul2(lo, p.rev ? make_float2(t.x, t.y) : make_float2(t.w, t.z));
            hi = mul2(hi, p.rev ? make_float2(t.z, t.w) : make_float2(t.y, t.x));
            pw[q][2 * e] = pack_bf16(lo.x, lo.y), pw[q][2 * e + 1] = pack_bf16(hi.x, hi.y);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const int lag = p.rev ? j0 + e - row : row - j0 - e;
            const bool on = lag >= 0 && j0 + e < m;  // select, not multiply: a later token may be NaN
            v[e] = on ? v[e] * (now ? s_pow[lag & 31] : ex2(l2 * (float)lag)) : 0.0f;
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) pw[q][e] = pack_bf16(v[2 * e], v[2 * e + 1]);
        }
      }
      if constexpr (NWG == 2) {  // all scores are read: P goes over them
        tc_fence_before();
        mbar_arrive(read);
        if (!(ok = wait_all(read, it))) break;
        tc_fence_after();
      }
#pragma unroll
      for (int q = 0; q < kBlocks; ++q) tmem_st16(tS + (half * kBlocks + q) * 16, pw[q]);
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(p_ready);
      // ---- y
      if (!(ok = wait_all(y_done, it))) break;
      tc_fence_after();
      const float lead = ex2(l2 * (float)(place + 1 - r)) * p.f;
      __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.y) + ((b * p.L + t0 + row) * p.H + h) * (int64_t)p.Dv;
      const bool wide = p.Dv % 16 == 0 && reinterpret_cast<uintptr_t>(p.y) % 32 == 0;  // rows of whole 32 bytes
#pragma unroll
      for (int c = 0; c < kYCols; c += 16) {
        float a[16], x[16];
        tmem_ld16_nowait(tY + y0 + c, a);
        tmem_ld16_nowait(tX + y0 + c, x);
        tmem_wait_ld();
        tmem_pin<16>(a);
        tmem_pin<16>(x);
        uint32_t q[8];
#pragma unroll
        for (int e = 0; e < 8; ++e)
          q[e] = pack_bf16(fmaf(lead, x[2 * e], p.f * a[2 * e]), fmaf(lead, x[2 * e + 1], p.f * a[2 * e + 1]));
        if (row < m && y0 + c < p.Dv) {
          if (wide) {
            store32(out + y0 + c, q);
          } else {
            *reinterpret_cast<uint4*>(out + y0 + c) = make_uint4(q[0], q[1], q[2], q[3]);
            if (y0 + c + 8 < p.Dv) *reinterpret_cast<uint4*>(out + y0 + c + 8) = make_uint4(q[4], q[5], q[6], q[7]);
          }
        }
      }
      tc_fence_before();
    }
    // ---- the final state, and zeros behind the length
    if (state_out && holds_t) {
      if (ok && chunks > 0) ok = wait_all(t_done, chunks - 1);
      tc_fence_after();
#pragma unroll 1
      for (int c = 0; c < kYCols && ok; c += 16) {
        float v[16];
        tmem_ld16_nowait(tT + y0 + c, v);
        tmem_wait_ld();
        tmem_pin<16>(v);
        if (row < p.Dk) {
          float* to = p.last + bh * sz + (int64_t)row * p.Dv + y0 + c;
#pragma unroll
          for (int e = 0; e < 16; e += 4)
            if (y0 + c + e < p.Dv) {
              float4 t = make_float4(p.last_f * v[e], p.last_f * v[e + 1], p.last_f * v[e + 2], p.last_f * v[e + 3]);
              *reinterpret_cast<float4*>(to + e) = t;
            }
        }
      }
    } else if (ok && chunks > 0) {
      wait_all(t_done, chunks - 1);  // no product is in flight when TMEM is given back
    }
    const int e8 = p.Dv / 8;
    for (int t = max(c_lo * kTok, n) + (tid >> 3); t < min(c_end * kTok, p.L); t += NWG * 16)
      for (int e = tid & 7; e < e8; e += 8)
        *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.y) + ((b * p.L + t) * p.H + h) * (int64_t)p.Dv + e * 8) =
            make_uint4(0, 0, 0, 0);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (s_abort) {  // the same for all: nothing writes it after the barrier
    if (warp == kMmaWarp) drain_umma(drain);
    if (warp == kTmaWarp && lane == 0) {
      drain_copies(xk_full, asked_xk, 1);
      drain_copies(v_full, asked_v, 1);
    }
    __syncthreads();
  }
  if (warp == kMmaWarp)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(Sh::kCols) : "memory");
}

// ---- the segments' own sums --------------------------------------------------------------------
// No x and no y: T = sum over the segment of k_j^T (w_j v_j), w_j to the segment's end, summed in TMEM from its first
// chunk to its last without being read.  Two stages of k, v and pieces.
template <int DX, int DY> struct SumShape {
  using Sh = Shape<DX, DY, 3>;
  static constexpr int kNP = 3;
  static constexpr int kStages = 2;
  static constexpr int kIn = Sh::kX + Sh::kV, kStage = kIn;
  // the pieces of one stage at a time where two do not fit
  static constexpr int kPieceSets = DX == 128 && DY == 128 ? 1 : 2;
  // with 64 dims the products read 64 rows behind an operand, for rows of the result that nobody reads
  static constexpr int kBehind = DX == 64 && !Sh::kScaleV ? kBlock : 0;
  static constexpr size_t kBytes = kStages * (size_t)kStage + kPieceSets * (size_t)kNP * Sh::kPiece + kBehind + 1024;
  static constexpr int kThreads = 128 + 64;
  static constexpr uint32_t kCols = DY;
  static constexpr int kBars = 2 * kStages + 2 + 2 + 2;
};

template <int DX, int DY>
__global__ void __launch_bounds__(SumShape<DX, DY>::kThreads, 1)
    sums_kernel(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
                const __grid_constant__ Pass p) {
  using Ss = SumShape<DX, DY>;
  using Sh = typename Ss::Sh;
  constexpr int NP = Ss::kNP, ST = Ss::kStages, PS = Ss::kPieceSets;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char *sIn = smem, *sP = smem + ST * Ss::kStage;
  __shared__ uint32_t s_tmem;
  __shared__ volatile int s_abort;
  __shared__ uint64_t bars[Ss::kBars];
  uint64_t *full = bars, *used = bars + ST, *ready = bars + 2 * ST, *taken = ready + 2, *done = taken + 1,
           *drain = done + 1;
  // used[s]: the products of stage s's chunk are complete; ready[i]: a chunk's pieces are written
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  constexpr int kTmaWarp = 4, kMmaWarp = 5;
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)),
                 "r"(Ss::kCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (tid == 0) {
    s_abort = 0;
    for (uint64_t* b = bars; b < bars + Ss::kBars; ++b) mbar_init(b, b >= ready && b < ready + 2 ? 128 : 1);
    fence_mbar_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_wait();
  pdl_trigger();
  const uint32_t tmem = s_tmem;
  const int seg = (int)(blockIdx.x % p.segs);
  const int64_t bh = blockIdx.x / p.segs, b = bh / p.H;
  const int h = (int)(bh - b * p.H);
  const int n = length(p, b);
  const float l2 = log2_decay(p.log_decay, h);
  const int lo = seg * p.seg_chunks * kTok, hi = min(min(lo + p.seg_chunks * kTok, p.L), n);
  const int chunks = hi > lo ? (hi - lo + kTok - 1) / kTok : 0;
  auto wait = [&](uint64_t* bar, uint32_t parity) { return mbar_wait_or(bar, parity & 1, &s_abort, p.err); };
  auto wait_all = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)) != 0; };
  int asked = 0;
  if (warp == kTmaWarp) {
    if (lane == 0)
      for (int it = 0; it < chunks; ++it) {
        const int s = it % ST, t0 = lo + it * kTok;
        if (it >= ST && !wait(&used[s], it / ST - 1)) break;
        mbar_expect_tx(&full[s], Ss::kIn);
        unsigned char* to = sIn + s * Ss::kStage;
        for (int d = 0; d < DX / 64; ++d) tma_load_4d(to + d * kBlock, &mk, d * 64, t0, h, (int)b, &full[s]);
        for (int d = 0; d < DY / 64; ++d) tma_load_4d(to + Sh::kX + d * kBlock, &mv, d * 64, t0, h, (int)b, &full[s]);
        asked = it + 1;
      }
  } else if (warp == kMmaWarp) {
    const uint32_t one = elect_one();
    const uint32_t id_t = idesc_bf16(128, (p.Dv + 15) / 16 * 16, true, true);
    const uint64_t d_k = smem_desc_sw128(smem_u32(sIn), kBlock, 1024),
                   d_v = smem_desc_sw128(smem_u32(sIn + Sh::kX), kBlock, 1024),
                   d_p = smem_desc_sw128(smem_u32(sP), kBlock, 1024);
    for (int it = 0; it < chunks; ++it) {
      const int s = it % ST, ps = it % PS;
      if (!wait_all(&ready[it & 1], it >> 1)) break;
      tc_fence_after();
#pragma unroll
      for (int i = 0; i < NP; ++i)
#pragma unroll
        for (int k = 0; k < kTok / 16; ++k) {
          const uint64_t pd = desc_at(d_p, (ps * NP + i) * Sh::kPiece + k * 16 * kRowBytes);
          const uint32_t off = s * Ss::kStage + k * 16 * kRowBytes;
          umma_ss(one, tmem, Sh::kScaleV ? desc_at(d_k, off) : pd, Sh::kScaleV ? pd : desc_at(d_v, off), id_t,
                  (it | i | k) != 0);
        }
      umma_done(one, &used[s]);
      if (it == chunks - 1) umma_done(one, done);
    }
  } else {
    const int row = tid & 127;
    constexpr int kPDims = Sh::kScaleV ? DY : DX;
    bool ok = true;
    for (int it = 0; it < chunks && ok; ++it) {
      const int s = it % ST, t = lo + it * kTok + row;
      // the products that read these pieces before
      if (it >= PS && !(ok = wait_all(&used[(it - PS) % ST], (it - PS) / ST))) break;
      if (!(ok = wait_all(&full[s], it / ST))) break;
      unsigned char *sK = sIn + s * Ss::kStage, *sV = sK + Sh::kX;
      if (t >= hi) {
        unsigned char* other = Sh::kScaleV ? sK : sV;
        for (int c = 0; c < (Sh::kScaleV ? DX : DY) / 8; ++c)
          *reinterpret_cast<uint4*>(other + swizzled(kTok, row, c)) = make_uint4(0, 0, 0, 0);
      }
      const float w = ex2(l2 * (float)(p.rev ? t - lo + 1 : hi - 1 - t));
      const unsigned char* from = Sh::kScaleV ? sV : sK;
      unsigned char* to = sP + it % PS * NP * Sh::kPiece;
#pragma unroll 2
      for (int c = 0; c < kPDims / 8; ++c) {
        const int at = swizzled(kTok, row, c);
        uint32_t q[NP][4] = {};
        if (t < hi) {
          const uint4 raw = *reinterpret_cast<const uint4*>(from + at);
          const uint32_t in[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float a = __uint_as_float(in[e] << 16) * w, z = __uint_as_float(in[e] & 0xffff0000u) * w;
#pragma unroll
            for (int i = 0; i < NP; ++i) {
              q[i][e] = pack_bf16(a, z);
              a -= __uint_as_float(q[i][e] << 16), z -= __uint_as_float(q[i][e] & 0xffff0000u);
            }
          }
        }
#pragma unroll
        for (int i = 0; i < NP; ++i)
          *reinterpret_cast<uint4*>(to + i * Sh::kPiece + at) = make_uint4(q[i][0], q[i][1], q[i][2], q[i][3]);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      mbar_arrive(&ready[it & 1]);
    }
    if (ok && chunks > 0) ok = wait_all(done, 0);
    tc_fence_after();
    if ((warp & 3) * 32 < DX) {
      float* to = p.part + (bh * p.segs + seg) * ((int64_t)p.Dk * p.Dv) + (int64_t)row * p.Dv;
      const uint32_t tT = tmem + ((uint32_t)((warp & 3) * 32) << 16);
#pragma unroll 1
      for (int c = 0; c < DY; c += 16) {
        float v[16] = {};
        if (chunks > 0) {
          tmem_ld16_nowait(tT + c, v);
          tmem_wait_ld();
          tmem_pin<16>(v);
        }
        if (row < p.Dk) {
#pragma unroll
          for (int e = 0; e < 16; e += 4)
            if (c + e < p.Dv) *reinterpret_cast<float4*>(to + c + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (s_abort) {
    if (warp == kMmaWarp) drain_umma(drain);
    if (warp == kTmaWarp && lane == 0) drain_copies(full, asked, ST);
    __syncthreads();
  }
  if (warp == kMmaWarp)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(Ss::kCols) : "memory");
}

// ---- host ----------------------------------------------------------------------------------
bool tc_ok(const Pass& p) {
  return p.Dk % 8 == 0 && p.Dv % 8 == 0 && mappable(p.x, p.L, p.H, p.B) && mappable(p.k, p.L, p.H, p.B) &&
         mappable(p.v, p.L, p.H, p.B) && reinterpret_cast<uintptr_t>(p.y) % 16 == 0 &&
         reinterpret_cast<uintptr_t>(p.last) % 16 == 0;
}

size_t tc_part_bytes(Pass p) {
  cut(p, kTok, 1);
  return p.segs > 1 ? (size_t)p.B * p.H * p.segs * p.Dk * p.Dv * sizeof(float) : 0;
}

template <int DX, int DY, int NP>
int launch(const Pass& p, cudaStream_t st) {
  using Sh = Shape<DX, DY, NP>;
  auto fn = tc_kernel<DX, DY, NP>;
  // before the maps: encoding one needs the device's context, which this call makes current in a new thread
  if (!set_smem_limit(reinterpret_cast<const void*>(fn), Sh::kBytes)) return HCLSM_ERR_LAUNCH;
  CUtensorMap mx, mk, mv;
  if (!make_map(&mx, p.x, p.Dk, p.L, p.H, p.B, kTok) || !make_map(&mk, p.k, p.Dk, p.L, p.H, p.B, kTok) ||
      !make_map(&mv, p.v, p.Dv, p.L, p.H, p.B, kTok))
    return HCLSM_ERR_UNSUPPORTED;
  const int64_t grid = (int64_t)p.B * p.H * p.segs;
  if (grid > 0x7fffffff) return HCLSM_ERR_SHAPE;
  if (p.segs > 1) {
    using Ss = SumShape<DX, DY>;
    auto sums = sums_kernel<DX, DY>;
    if (!set_smem_limit(reinterpret_cast<const void*>(sums), Ss::kBytes)) return HCLSM_ERR_LAUNCH;
    if (const int rc = launch_pdl(sums, (unsigned)grid, Ss::kThreads, Ss::kBytes, st, mk, mv, p)) return rc;
    if (const int rc = join(p, kTok, st)) return rc;
  }
  return launch_pdl(fn, (unsigned)grid, Sh::kThreads, Sh::kBytes, st, mx, mk, mv, p);
}

template <int DX, int DY>
int launch_np(const Pass& p, cudaStream_t st) {
  return p.last && p.segs == 1 ? launch<DX, DY, 3>(p, st) : launch<DX, DY, 2>(p, st);
}

int tc_pass(Pass p, cudaStream_t st) {
  cut(p, kTok, 1);
  if (p.Dk <= 64) return p.Dv <= 64 ? launch_np<64, 64>(p, st) : launch_np<64, 128>(p, st);
  return p.Dv <= 64 ? launch_np<128, 64>(p, st) : launch_np<128, 128>(p, st);
}

}  // namespace decay
}  // namespace hclsm
