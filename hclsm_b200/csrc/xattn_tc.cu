// Cross attention in bf16 on the 5th-generation tensor cores (tcgen05, TMEM, TMA).
//
// Forward: a block takes QT tiles of 128 query rows of one head (QT 2: one block
// an SM; QT 1: two), each with a softmax warpgroup (thread = row = TMEM lane), a warp
// that issues TMA and one or two that issue MMA.  Per tile of 128 keys:
//   S = Q K^T        128 x 128, fp32 in TMEM
//   the row's thread reads its scores, takes the running maximum, writes
//   P = exp2(c s - m) as bf16 to TMEM, keeps the row's sum in fp32
//   O += P V         A from TMEM, V as the MN-major B operand; fp32 in TMEM
// The maximum that O is scaled by is raised only when a row's new one exceeds it by
// 8 (in log2): until then the weights are at most 2^8, which fp32 and bf16 hold
// with the same relative precision, and O is read back and rescaled rarely.
// The bound is the softmax's issue and its chain with the products: 4 x 2048 queries
// over 8192 states, 32 heads of 64, 690 to 700 us (785 to 797 TFLOP/s), 8 x 2048 over 4096, 16
// heads of 128, 435 to 474 us (1160 to 1264 TFLOP/s, by the clock); tensor pipe 28 and 44 % busy (2 x 2048
// over 4096).
// While one tile takes its softmax the tensor cores run the other's products.
#include "xattn_tc.cuh"

namespace hclsm {
namespace xattn {

constexpr float kRaise = 8.0f;

template <int DP, int QT> struct FwdShape {
  static constexpr int kBlock = kTile * kRowBytes;        // 64 dims of a tile
  static constexpr int kOp = DP / 64 * kBlock;            // a staged tile
  static constexpr int kStages = DP == 64 ? (QT == 2 ? 3 : 2) : (QT == 2 ? 2 : 1);
  // D <= 64 leaves TMEM columns for the weights beside the scores: then the next tile's
  // scores are formed as soon as this tile's have been read.  Else the weights go over
  // the scores; so with QT 1, whose second block an SM hides the wait, and where a third
  // warp of issue would cost the softmax threads 40 registers (spills).
  static constexpr bool kApart = DP == 64 && QT == 2;
  static constexpr int kBars = 1 + 4 * kStages + 4 * QT + 2;
  static constexpr int kColP = kApart ? QT * 128 : 0, kColO = QT * (kApart ? 192 : 128);
  static constexpr int kStepP = kApart ? 64 : 128;  // columns from one tile's weights to the next's
  static constexpr size_t kBytes = (size_t)(QT + 2 * kStages) * kOp + kBars * 8 + 1024;
  static constexpr int kThreads = QT * 128 + (kApart ? 96 : 64);
  static constexpr uint32_t kCols = QT == 2 ? 512 : 256;
};

template <int DP, int QT>
__global__ void __launch_bounds__(FwdShape<DP, QT>::kThreads, QT == 1 ? 2 : 1)
    tc_fwd_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                  const __grid_constant__ CUtensorMap mv, const __grid_constant__ TcParams p) {
  using Sh = FwdShape<DP, QT>;
  constexpr int ST = Sh::kStages;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint32_t s_tmem;
  __shared__ volatile int s_abort;
  unsigned char *sQ = smem, *sK = sQ + QT * Sh::kOp, *sV = sK + ST * Sh::kOp;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sV + ST * Sh::kOp);
  uint64_t *q_full = bars, *k_full = bars + 1, *k_empty = k_full + ST, *v_full = k_empty + ST, *v_empty = v_full + ST,
           *s_full = v_empty + ST, *p_full = s_full + QT, *pv_done = p_full + QT, *s_free = pv_done + QT,
           *drain = s_free + QT;
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  constexpr int kTmaWarp = QT * 4, kMmaWarp = QT * 4 + 1, kWeighWarp = QT * 4 + 2;
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)),
                 "r"(Sh::kCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  const int q0 = (int)(blockIdx.x % p.qtiles) * (QT * kTile);
  if (tid == 0) {
    s_abort = 0;
    // Warps without a row take no part in the tiles' phases: with the weights apart from the scores, one that only
    // arrived could be a whole tile ahead of a warp still at its last weights and end that warp's phase for it.
    auto rows = [&](int w) {  // threads of query tile w's warps that have a row (a count is at least 1)
      const int n = p.x.Lq - q0 - w * kTile;
      return n >= kTile ? kTile : n > 0 ? (n + 31) / 32 * 32 : 1;
    };
    for (uint64_t* bar = bars; bar < bars + Sh::kBars; ++bar) {
      const int w = bar >= p_full && bar < pv_done ? (int)(bar - p_full)
                    : bar >= s_free && bar < drain ? (int)(bar - s_free)
                                                   : -1;
      mbar_init(bar, w >= 0 ? rows(w) : 1);
    }
    fence_mbar_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_wait();
  pdl_trigger();
  // tile w: scores in columns [w * 128, + 128), weights in [kColP + w * kStepP, + 64), O in [kColO + w * DP, + DP)
  const uint32_t tmem = s_tmem;
  const Params& x = p.x;
  const int h = (int)(blockIdx.x / p.qtiles % x.H), hk = h / (x.H / x.Hkv);
  const int64_t b = blockIdx.x / p.qtiles / x.H;
  const int nk = key_count(x, b), tiles = (nk + kTile - 1) / kTile;
  const int nq = QT == 2 && q0 + kTile >= x.Lq ? 1 : QT;  // tiles with rows
  auto wait = [&](uint64_t* bar, uint32_t parity) { return mbar_wait_or(bar, parity & 1, &s_abort, x.err); };
  // the whole warp goes on or gives up together
  auto wait_all = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)) != 0; };

  int issued = 0;  // copies of K and of V (lane 0 of the TMA warp)
  if (warp == kTmaWarp) {
    if (lane == 0 && tiles > 0) {
      mbar_expect_tx(q_full, nq * Sh::kOp);
      for (int w = 0; w < nq; ++w)
        for (int kb = 0; kb < DP / 64; ++kb)
          tma_load_4d(sQ + w * Sh::kOp + kb * Sh::kBlock, &mq, kb * 64, q0 + w * kTile, h, (int)b, q_full);
      for (int j = 0; j < tiles; ++j) {
        const int s = j % ST;
        const uint32_t ph = j / ST;
        if (!wait(&k_empty[s], ph ^ 1)) break;
        mbar_expect_tx(&k_full[s], Sh::kOp);
        for (int kb = 0; kb < DP / 64; ++kb)
          tma_load_4d(sK + s * Sh::kOp + kb * Sh::kBlock, &mk, kb * 64, j * kTile, hk, (int)b, &k_full[s]);
        if (!wait(&v_empty[s], ph ^ 1)) {
          mbar_wait(&k_full[s], ph & 1);  // given up: the K just asked for arrives first
          break;
        }
        mbar_expect_tx(&v_full[s], Sh::kOp);
        for (int kb = 0; kb < DP / 64; ++kb)
          tma_load_4d(sV + s * Sh::kOp + kb * Sh::kBlock, &mv, kb * 64, j * kTile, hk, (int)b, &v_full[s]);
        issued = j + 1;
      }
    }
  } else if (warp == kMmaWarp || warp == kWeighWarp) {
    const uint32_t id_s = idesc_bf16(kTile, kTile, false, false);
    const uint32_t id_o = idesc_bf16(kTile, (x.D + 15) / 16 * 16, false, true);
    const int ksteps = (x.D + 15) / 16;
    const uint64_t d_q = smem_desc_sw128(smem_u32(sQ), 16, 1024), d_k = smem_desc_sw128(smem_u32(sK), 16, 1024),
                   d_v = smem_desc_sw128(smem_u32(sV), Sh::kBlock, 1024);
    const uint32_t one = elect_one();
    auto scores = [&](int w, int s) {
      const uint64_t a = desc_at(d_q, w * Sh::kOp), bk = desc_at(d_k, s * Sh::kOp);
#pragma unroll
      for (int k = 0; k < DP / 16; ++k) {
        const uint32_t off = (k >> 2) * Sh::kBlock + (k & 3) * 32;
        if (k < ksteps) umma_ss(one, tmem + w * 128, desc_at(a, off), desc_at(bk, off), id_s, k != 0);
      }
      umma_done(one, &s_full[w]);
    };
    auto weigh = [&](int w, int j) {  // O of tile w += its weights of keys j times V
      const uint64_t bv = desc_at(d_v, j % ST * Sh::kOp);
#pragma unroll
      for (int k = 0; k < kTile / 16; ++k)
        umma_ts(one, tmem + Sh::kColO + w * DP, tmem + Sh::kColP + w * Sh::kStepP + k * 8,
                desc_at(bv, k * 16 * kRowBytes), id_o, (j | k) != 0);
      umma_done(one, &pv_done[w]);
      if (w == nq - 1) umma_done(one, &v_empty[j % ST]);
    };
    auto values = [&](int j) {  // V of keys j is there, and zero where it is not allowed
      if (!wait_all(&v_full[j % ST], j / ST)) return false;
      const uint4 bits = key_bits(p, b, nk, j * kTile);
      if (!all_bits(bits)) zero_rows<DP, kTile>(sV + j % ST * Sh::kOp, bits, lane);
      return true;
    };
    bool ok = tiles > 0;
    if constexpr (Sh::kApart) {
      // Scores and weighted sums wait for different threads: a warp issues each, so that
      // neither waits behind the other.
      if (warp == kMmaWarp) {
        ok = ok && wait_all(q_full, 0);
        for (int j = 0; j < tiles && ok; ++j) {
          const int s = j % ST;
          if (!(ok = wait_all(&k_full[s], j / ST))) break;
          for (int w = 0; w < nq && ok; ++w) {
            if (j > 0 && !(ok = wait_all(&s_free[w], j - 1))) break;
            tc_fence_after();
            scores(w, s);
          }
          if (ok) umma_done(one, &k_empty[s]);
        }
      } else {
        for (int j = 0; j < tiles && ok; ++j) {
          if (!(ok = values(j))) break;
          for (int w = 0; w < nq && ok; ++w) {
            if (!(ok = wait_all(&p_full[w], j))) break;
            tc_fence_after();
            weigh(w, j);
          }
        }
      }
    } else if (warp == kMmaWarp) {
      ok = ok && wait_all(q_full, 0) && wait_all(&k_full[0], 0);
      if (ok) {
        tc_fence_after();
        for (int w = 0; w < nq; ++w) scores(w, 0);
        umma_done(one, &k_empty[0]);
      }
      for (int j = 0; j < tiles && ok; ++j) {
        const int s1 = (j + 1) % ST;
        if (!(ok = values(j))) break;
        for (int w = 0; w < nq && ok; ++w) {
          if (!(ok = wait_all(&p_full[w], j))) break;
          tc_fence_after();
          weigh(w, j);
          if (j + 1 < tiles) {
            if (w == 0 && !(ok = wait_all(&k_full[s1], (j + 1) / ST))) break;
            tc_fence_after();
            scores(w, s1);
            if (w == nq - 1) umma_done(one, &k_empty[s1]);
          }
        }
      }
    }
  } else {
    const int w = warp >> 2;
    const int row = q0 + w * kTile + (tid & 127);
    const bool idle = q0 + w * kTile + (warp & 3) * 32 >= x.Lq;  // no row of this warp
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + lanes + w * 128, tP = tmem + lanes + Sh::kColP + w * Sh::kStepP,
                   tO = tmem + lanes + Sh::kColO + w * DP;
    const float c2 = x.scale * kLog2e;
    float m = -INFINITY;  // the maximum O is scaled by, raw scores
    float2 l = make_float2(0.0f, 0.0f);
    bool ok = !idle;
    for (int j = 0; j < tiles && ok; ++j) {
      const uint4 bits = key_bits(p, b, nk, j * kTile);
      if (!(ok = wait_all(&s_full[w], j))) break;
      tc_fence_after();
      if (!all_bits(bits)) {  // -inf over the scores that do not count; the rest of the code has no mask
#pragma unroll 1
        for (int c = 0; c < 8; ++c) {
          const uint32_t word = (c < 4 ? (c < 2 ? bits.x : bits.y) : (c < 6 ? bits.z : bits.w)) >> (16 * (c & 1));
          float v[16];
          tmem_ld16_nowait(tS + c * 16, v);
          tmem_wait_ld();
          tmem_pin<16>(v);
          uint32_t q[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) q[i] = word >> i & 1u ? __float_as_uint(v[i]) : 0xff800000u;
          tmem_st16(tS + c * 16, q);
        }
        tmem_wait_st();
      }
      auto highest = [&](float (&mx)[4], const float (&v)[32]) {
#pragma unroll
        for (int i = 0; i < 32; i += 8)
#pragma unroll
          for (int q = 0; q < 4; ++q) mx[q] = max3(mx[q], v[i + q], v[i + q + 4]);
      };
      // a row's maximum is now `top`: O, kept by the old one, is scaled to it where it is too low
      auto raise = [&](float top) {
        const bool up = (top - m) * c2 > kRaise;  // false where both are -inf (NaN)
        if (!__any_sync(0xffffffffu, up)) return;
        const float f = up ? ex2((m - top) * c2) : 1.0f;  // 0 from -inf: O is zero, or (j = 0) not yet written
        if (up) m = top;
        l.x *= f, l.y *= f;
        if (j > 0) {
          ok = wait_all(&pv_done[w], j - 1);
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < DP && ok; c += 16) {
            float o[16];
            tmem_ld16_nowait(tO + c, o);
            tmem_wait_ld();
            tmem_pin<16>(o);
            uint32_t q[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) q[i] = __float_as_uint(o[i] * f);
            tmem_st16(tO + c, q);
          }
        }
      };
      // 32 scores to weights; three pairs in eight on the FMA pipe, because the MUFU's 16 a clock
      // would be the bound (measured for a 128 x 128 tile of two warpgroups: 1196 clocks with
      // none there, 1071 with two in eight, 1003 with three, 1061 with four)
      auto weights = [&](const float (&v)[32], uint32_t* pw, float2& sum) {
        const float base = m == -INFINITY ? 0.0f : -m * c2;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float2 e = fma2(make_float2(v[2 * i], v[2 * i + 1]), make_float2(c2, c2), make_float2(base, base));
          if (0xa8 >> (i & 7) & 1) e = ex2_fma(e);
          else e.x = ex2(e.x), e.y = ex2(e.y);
          sum = add2(sum, e);
          pw[i] = pack_bf16(e.x, e.y);
        }
      };
      // fn(chunk, its 32 scores), each chunk's load in flight during the one before
      auto chunks = [&](auto fn) {
        float v[2][32];
        tmem_ld32_nowait(tS, v[0]);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          tmem_wait_ld();
          tmem_pin<32>(v[c & 1]);
          if (c < 3) tmem_ld32_nowait(tS + (c + 1) * 32, v[(c + 1) & 1]);
          fn(c, v[c & 1]);
        }
      };
      // The maximum first, then the weights from a second reading: a row's scores and weights
      // together do not fit the registers (weights by the old maximum, kept until the new one
      // is known, took 481 against 435 us with heads of 128, spills included).
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      chunks([&](int, const float (&v)[32]) { highest(mx, v); });
      raise(max3(fmaxf(mx[0], mx[1]), mx[2], mx[3]));
      if constexpr (Sh::kApart) {
        if (ok && j > 0) ok = wait_all(&pv_done[w], j - 1);  // the last weights have been used
        tc_fence_after();
      }
      if (!ok) break;
      float2 sum = make_float2(0.0f, 0.0f);
      chunks([&](int c, const float (&v)[32]) {
        if (Sh::kApart && c == 3) {  // the scores are free while their last quarter is still being weighed
          tc_fence_before();
          mbar_arrive(&s_free[w]);
        }
        uint32_t pw[16];
        weights(v, pw, sum);
        tmem_st16(tP + c * 16, pw);  // where over the scores: over ones that have been read
      });
      l = add2(l, sum);
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&p_full[w]);
    }
    if (ok && tiles > 0) ok = wait_all(&pv_done[w], tiles - 1);
    tc_fence_after();
    if (!idle) {
      const float sum = l.x + l.y;
      const float inv = tiles > 0 && sum != 0.0f ? 1.0f / sum : 0.0f;
      if (row < x.Lq && x.lse2) x.lse2[(b * x.H + h) * x.Lq + row] = sum == 0.0f ? INFINITY : m * c2 + log2f(sum);
      __nv_bfloat16* out = static_cast<__nv_bfloat16*>(x.o) + ((b * x.Lq + row) * x.H + h) * (int64_t)x.D;
#pragma unroll
      for (int c = 0; c < DP; c += 32) {
        float o[32];
        if (tiles > 0) {
          tmem_ld32_nowait(tO + c, o);
          tmem_wait_ld();
          tmem_pin<32>(o);
        }
        if (row < x.Lq) {
#pragma unroll
          for (int i = 0; i < 32; i += 8)
            if (c + i < x.D) {
              uint32_t q[4];
#pragma unroll
              for (int e = 0; e < 4; ++e)  // a row without keys: zero, whatever O holds
                q[e] = inv == 0.0f ? 0u : pack_bf16(o[i + 2 * e] * inv, o[i + 2 * e + 1] * inv);
              *reinterpret_cast<uint4*>(out + c + i) = make_uint4(q[0], q[1], q[2], q[3]);
              if (x.lo) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  q[e] = inv == 0.0f ? 0u : pack_bf16(rounding(o[i + 2 * e] * inv), rounding(o[i + 2 * e + 1] * inv));
                *reinterpret_cast<uint4*>(x.lo + (out - static_cast<__nv_bfloat16*>(x.o)) + c + i) =
                    make_uint4(q[0], q[1], q[2], q[3]);
              }
            }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (s_abort) {  // the same for all: nothing writes it after the barrier
    if (warp == kMmaWarp || warp == kWeighWarp) drain_umma(&drain[warp - kMmaWarp]);
    if (warp == kTmaWarp && lane == 0 && tiles > 0) {
      mbar_wait(q_full, 0);
      drain_copies(k_full, issued, ST);
      drain_copies(v_full, issued, ST);
    }
    __syncthreads();
  }
  if (warp == kMmaWarp)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(Sh::kCols) : "memory");
}

// ---- the key mask as bits ------------------------------------------------------------------
__global__ void __launch_bounds__(256) bits_kernel(const __grid_constant__ Params p, uint32_t* words, int word_sb) {
  pdl_wait();
  pdl_trigger();
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t b = i / ((int64_t)word_sb * 32);
  const int j = (int)(i % ((int64_t)word_sb * 32));
  const bool on = b < p.B && j < p.Lk && p.mask[b * p.mask_sb + j];
  const uint32_t w = __ballot_sync(0xffffffffu, on);
  if ((threadIdx.x & 31) == 0 && b < p.B) words[b * word_sb + j / 32] = w;
}

bool tc_ok(const Params& p, bool bwd) {
  return p.D % 8 == 0 && p.Lk > 0 && p.Lq > 0 && mappable(p.q, p.Lq, p.H, p.B) && mappable(p.k, p.Lk, p.Hkv, p.B) &&
         mappable(p.v, p.Lk, p.Hkv, p.B) && (!bwd || mappable(p.dout, p.Lq, p.H, p.B)) &&
         reinterpret_cast<uintptr_t>(p.o) % 16 == 0;
}

size_t tc_workspace(const Params& p) { return p.mask ? (size_t)p.B * word_stride(p) * sizeof(uint32_t) : 0; }

int make_bits(TcParams& t, void* ws, cudaStream_t st) {
  t.words = nullptr, t.word_sb = 0;
  if (!t.x.mask) return HCLSM_OK;
  t.word_sb = word_stride(t.x);
  t.words = static_cast<uint32_t*>(ws);
  const int64_t grid = ((int64_t)t.x.B * t.word_sb * 32 + 255) / 256;
  if (grid > 0x7fffffff) return HCLSM_ERR_SHAPE;
  return launch_pdl(bits_kernel, (unsigned)grid, 256, 0, st, t.x, static_cast<uint32_t*>(ws), t.word_sb);
}

template <int DP, int QT>
static int launch_fwd(TcParams& t, cudaStream_t st) {
  using Sh = FwdShape<DP, QT>;
  const Params& x = t.x;
  // before the maps: encoding one needs the device's context, which this call makes current in a new thread
  auto fn = tc_fwd_kernel<DP, QT>;
  if (!set_smem_limit(reinterpret_cast<const void*>(fn), Sh::kBytes)) return HCLSM_ERR_LAUNCH;
  CUtensorMap mq, mk, mv;
  if (!make_map(&mq, x.q, x.D, x.Lq, x.H, x.B, kTile) || !make_map(&mk, x.k, x.D, x.Lk, x.Hkv, x.B, kTile) ||
      !make_map(&mv, x.v, x.D, x.Lk, x.Hkv, x.B, kTile))
    return HCLSM_ERR_UNSUPPORTED;
  t.qtiles = (x.Lq + QT * kTile - 1) / (QT * kTile);
  const int64_t grid = (int64_t)t.qtiles * x.H * x.B;
  if (grid > 0x7fffffff) return HCLSM_ERR_SHAPE;
  return launch_pdl(fn, (unsigned)grid, Sh::kThreads, Sh::kBytes, st, mq, mk, mv, t);
}

int tc_fwd(const Params& p, void* ws, cudaStream_t st) {
  TcParams t = {};
  t.x = p;
  if (const int rc = make_bits(t, ws, st)) return rc;
  const bool two = p.Lq > kTile;
  if (p.D <= 64) return two ? launch_fwd<64, 2>(t, st) : launch_fwd<64, 1>(t, st);
  return two ? launch_fwd<128, 2>(t, st) : launch_fwd<128, 1>(t, st);
}

}  // namespace xattn
}  // namespace hclsm
