// Cross attention backward in bf16 on the 5th-generation tensor cores.
//
// Two kernels, each with its own recomputation of the weights, so that every sum
// has a fixed order (no atomics): 7 products instead of 5.
//
//   dq: a block takes 128 query rows (q and do as A operands in TMEM; delta on the way)
//   and walks over tiles of 64 keys:
//     S = Q K^T, dP = dO V^T  ->  dS = P (dP - delta), bf16 over S  ->  dQ += dS K
//   dk, dv: a block takes 128 keys and walks over tiles of 64 query rows of every
//   query head that shares them, transposed so that keys are the TMEM lanes:
//     S^T = K Q^T, dP^T = V dO^T  ->  P^T over S^T, dS^T over dP^T  ->
//     dV += P^T dO, dK += dS^T Q
//
// The weights and their gradients are A operands in TMEM; the same staged tile of
// K (or Q, dO) is the K-major operand of one product and the MN-major operand of
// another.  Two buffers of 64 + 64 columns with warpgroups of their own: the tensor
// cores form one buffer's products while the other's weights are computed.  A tile of
// 64 and not 128: 2 x (128 + 128) columns and the accumulators (128 or 256) do not fit
// TMEM's 512.  4 x 2048 queries over 4096 states, 32 heads of 64: 1269 us.
// 8 x 2048 queries over 4096 states, 16 heads of 128 over 4: 1525 to 1565 us, of it 46 %
// for dq (3 products: 1150 TFLOP/s) and 54 % for dk and dv (4: 1300);
// the tensor pipe is 45 and 56 % busy (2 x 2048 over 4096).  What bounds it is the chain
// of products, weights and products; and in the second kernel 128 x 64 products with both
// operands in shared memory, 51 cycles a step of 16 instead of 35.
#include "xattn_tc.cuh"

namespace hclsm {
namespace xattn {

constexpr int kB = 64;  // keys (dq) or queries (dk, dv) of a streamed tile

template <int DP> struct BwdShape {
  static constexpr int kBlockA = kTile * kRowBytes, kBlockB = kB * kRowBytes;  // 64 dims
  static constexpr int kOpA = DP / 64 * kBlockA, kOpB = DP / 64 * kBlockB;
  static constexpr int kStages = 4;
  static constexpr int kBars = 1 + 2 * kStages + 4 + 2;
  // shared memory: dq has no own operands there
  static constexpr size_t kDqBytes = 2 * kStages * (size_t)kOpB + kBars * 8 + 1024, kDkvBytes = kDqBytes + 2 * kOpA;
  // Warpgroups a buffer: dq two (thread = half a row), dk and dv one (thread = row, whose
  // two results of 64 columns would spill the 96 registers that four warpgroups have).
  // 8 x 2048 x 4096, 16 heads of 128: dq 864 us with one, 740 with two; dk, dv 840 with
  // one, 1150 with two.
  static constexpr int kDqThreads = 4 * 128 + 64, kDkvThreads = 2 * 128 + 64;
};

// Shared by the two kernels: block layout, barriers, roles.  OWN: the block's own operands are in shared memory.
template <int DP, bool OWN> struct Block {
  using Sh = BwdShape<DP>;
  unsigned char *a0, *a1, *b0, *b1;  // the block's own two operands, the streamed two
  uint64_t *own, *full, *empty, *sd_full, *ds_full, *done, *drain;
  __device__ __forceinline__ explicit Block(unsigned char* raw) {
    a0 = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    a1 = a0 + (OWN ? Sh::kOpA : 0), b0 = a1 + (OWN ? Sh::kOpA : 0), b1 = b0 + Sh::kStages * Sh::kOpB;
    own = reinterpret_cast<uint64_t*>(b1 + Sh::kStages * Sh::kOpB);
    full = own + 1, empty = full + Sh::kStages, sd_full = empty + Sh::kStages, ds_full = sd_full + 2,
    done = ds_full + 2, drain = done + 1;
  }
  __device__ __forceinline__ void init(int threads) const {  // of a buffer
    for (int i = 0; i < Sh::kBars; ++i)
      mbar_init(own + i, own + i >= ds_full && own + i < done ? threads : !OWN && i == 0 ? 2 * threads : 1);
    fence_mbar_init();
  }
  // What the issuing thread computes once.
  struct Issue {
    uint64_t a0, a1, b0, b1, t0, t1;  // the operands K-major; the streamed two MN-major
    uint32_t id_s, id_o, one;
    int ksteps;
  };
  __device__ __forceinline__ Issue issue(int D) const {
    Issue r;
    r.one = elect_one();
    r.a0 = smem_desc_sw128(smem_u32(a0), 16, 1024), r.a1 = smem_desc_sw128(smem_u32(a1), 16, 1024);
    r.b0 = smem_desc_sw128(smem_u32(b0), 16, 1024), r.b1 = smem_desc_sw128(smem_u32(b1), 16, 1024);
    r.t0 = smem_desc_sw128(smem_u32(b0), Sh::kBlockB, 1024), r.t1 = smem_desc_sw128(smem_u32(b1), Sh::kBlockB, 1024);
    r.id_s = idesc_bf16(kTile, kB, false, false);
    r.id_o = idesc_bf16(kTile, (D + 15) / 16 * 16, false, true);
    r.ksteps = (D + 15) / 16;
    return r;
  }
  // buffer w's two products of the streamed tile in stage s (a converged warp)
  __device__ __forceinline__ void products(const Issue& r, uint32_t tmem, int w, int s) const {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const uint64_t b = desc_at(half ? r.b1 : r.b0, s * Sh::kOpB);
#pragma unroll
      for (int k = 0; k < DP / 16; ++k) {
        const uint32_t ka = (k >> 2) * Sh::kBlockA + (k & 3) * 32, kb = (k >> 2) * Sh::kBlockB + (k & 3) * 32;
        if (k < r.ksteps)
          umma_ss(r.one, tmem + w * 128 + half * 64, desc_at(half ? r.a1 : r.a0, ka), desc_at(b, kb), r.id_s, k != 0);
      }
    }
    umma_done(r.one, &sd_full[w]);
  }
  // the same with the own operands in TMEM columns t0 and t1
  __device__ __forceinline__ void products_ts(const Issue& r, uint32_t tmem, uint32_t t0, uint32_t t1, int w,
                                              int s) const {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const uint64_t b = desc_at(half ? r.b1 : r.b0, s * Sh::kOpB);
#pragma unroll
      for (int k = 0; k < DP / 16; ++k)
        if (k < r.ksteps)
          umma_ts(r.one, tmem + w * 128 + half * 64, (half ? t1 : t0) + k * 8,
                  desc_at(b, (k >> 2) * Sh::kBlockB + (k & 3) * 32), r.id_s, k != 0);
    }
    umma_done(r.one, &sd_full[w]);
  }
  // acc += (bf16 columns at a, the second 32 rows' STEP further) x (streamed tile in stage s, MN-major descriptor t)
  // (a converged warp)
  template <int STEP>
  __device__ __forceinline__ void accumulate(const Issue& r, uint32_t acc, uint32_t a, uint64_t t, int s,
                                             bool first) const {
    const uint64_t b = desc_at(t, s * Sh::kOpB);
#pragma unroll
    for (int k = 0; k < kB / 16; ++k)
      umma_ts(r.one, acc, a + (k & 1) * 8 + (k >> 1) * STEP, desc_at(b, k * 16 * kRowBytes), r.id_o,
              !(first && k == 0));
  }
};

__device__ __forceinline__ void alloc_tmem(uint32_t* slot) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(slot)) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void free_tmem(uint32_t tmem) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

// Columns [c0, c0 + n) of an accumulator's row to global memory, times f.
template <int N>
__device__ __forceinline__ void store_acc(uint32_t t, __nv_bfloat16* out, bool ok, bool zero, int c0, int D, float f) {
#pragma unroll
  for (int c = 0; c < N; c += 16) {
    float o[16];
    if (!zero) {
      tmem_ld16_nowait(t + c0 + c, o);
      tmem_wait_ld();
      tmem_pin<16>(o);
    }
    if (!ok) continue;
#pragma unroll
    for (int i = 0; i < 16; i += 8)
      if (c0 + c + i < D) {
        uint32_t r[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = zero ? 0u : pack_bf16(o[i + 2 * e] * f, o[i + 2 * e + 1] * f);
        *reinterpret_cast<uint4*>(out + c0 + c + i) = make_uint4(r[0], r[1], r[2], r[3]);
      }
  }
}

template <int DP>
__global__ void __launch_bounds__(BwdShape<DP>::kDqThreads, 1)
    tc_dq_kernel(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
                 const __grid_constant__ TcParams p) {
  using Sh = BwdShape<DP>;
  extern __shared__ unsigned char smem_raw[];
  __shared__ uint32_t s_tmem;
  __shared__ volatile int s_abort;
  __shared__ float s_delta[2][kTile];
  const Block<DP, false> blk(smem_raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  constexpr int kTmaWarp = 16, kMmaWarp = 17;
  if (warp == kMmaWarp) alloc_tmem(&s_tmem);
  if (tid == 0) {
    s_abort = 0;
    blk.init(256);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_wait();
  pdl_trigger();
  const uint32_t tmem = s_tmem, acc = tmem + 256, t_q = acc + DP, t_do = t_q + DP / 2;
  const Params& x = p.x;
  const int q0 = (int)(blockIdx.x % p.qtiles) * kTile;
  const int h = (int)(blockIdx.x / p.qtiles % x.H), hk = h / (x.H / x.Hkv);
  const int64_t b = blockIdx.x / p.qtiles / x.H;
  const int nk = key_count(x, b), tiles = (nk + kB - 1) / kB;
  auto wait = [&](uint64_t* bar, uint32_t parity) { return mbar_wait_or(bar, parity & 1, &s_abort, x.err); };
  // the whole warp goes on or gives up together
  auto wait_all = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)) != 0; };

  int issued = 0;  // streamed tiles asked for (lane 0 of the TMA warp)
  if (warp == kTmaWarp) {
    if (lane == 0 && tiles > 0) {
      for (int j = 0; j < tiles; ++j) {
        const int s = j % Sh::kStages;
        if (!wait(&blk.empty[s], j / Sh::kStages ^ 1)) break;
        mbar_expect_tx(&blk.full[s], 2 * Sh::kOpB);
        for (int kb = 0; kb < DP / 64; ++kb) {
          tma_load_4d(blk.b0 + s * Sh::kOpB + kb * Sh::kBlockB, &mk, kb * 64, j * kB, hk, (int)b, &blk.full[s]);
          tma_load_4d(blk.b1 + s * Sh::kOpB + kb * Sh::kBlockB, &mv, kb * 64, j * kB, hk, (int)b, &blk.full[s]);
        }
        issued = j + 1;
      }
    }
  } else if (warp == kMmaWarp) {
    const auto is = blk.issue(x.D);
    auto start = [&](int j) {  // the products of tile j into buffer j & 1
      const int s = j % Sh::kStages;
      if (!wait_all(&blk.full[s], j / Sh::kStages)) return false;
      const uint4 bits = key_bits(p, b, nk, j * kB & ~127);
      const uint4 mine = j & 1 ? make_uint4(bits.z, bits.w, ~0u, ~0u) : make_uint4(bits.x, bits.y, ~0u, ~0u);
      if (!all_bits(mine)) zero_rows<DP, kB>(blk.b0 + s * Sh::kOpB, mine, lane);  // dS 0 times K
      tc_fence_after();
      blk.products_ts(is, tmem, t_q, t_do, j & 1, s);
      return true;
    };
    bool ok = tiles > 0 && wait_all(blk.own, 0) && start(0) && (tiles < 2 || start(1));
    for (int j = 0; j < tiles && ok; ++j) {
      if (!(ok = wait_all(&blk.ds_full[j & 1], j >> 1))) break;
      tc_fence_after();
      const int s = j % Sh::kStages;
      blk.template accumulate<32>(is, acc, tmem + (j & 1) * 128, is.t0, s, j == 0);
      umma_done(is.one, &blk.empty[s]);
      if (j == tiles - 1) umma_done(is.one, blk.done);
      if (j + 2 < tiles) ok = start(j + 2);
    }
  } else {
    const int w = warp >> 3, half = warp >> 2 & 1;
    const int row = q0 + (tid & 127);
    const bool idle = q0 + (warp & 3) * 32 >= x.Lq;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + lanes + w * 128;
    const int64_t at = (b * x.H + h) * x.Lq + row;
    const float c2 = x.scale * kLog2e;
    // The block's own operands: buffer 0's threads bring q to TMEM, buffer 1's do, half a row each (zeros past the
    // ends), and take delta = do . o from it.
    {
      const View& src = w ? x.dout : x.q;
      const __nv_bfloat16* from =
          static_cast<const __nv_bfloat16*>(src.p) + b * src.sb + (int64_t)row * src.st + (int64_t)h * src.sh;
      const __nv_bfloat16* o = static_cast<const __nv_bfloat16*>(x.o) + ((b * x.Lq + row) * x.H + h) * (int64_t)x.D;
      float2 dot = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int c = 0; c < DP / 2; c += 32) {
        uint32_t r[16];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int d = half * (DP / 2) + c + i * 8;
          uint4 v = make_uint4(0, 0, 0, 0), u = v;
          if (row < x.Lq && d < x.D) {
            v = *reinterpret_cast<const uint4*>(from + d);
            if (w) u = *reinterpret_cast<const uint4*>(o + d);
          }
          r[4 * i] = v.x, r[4 * i + 1] = v.y, r[4 * i + 2] = v.z, r[4 * i + 3] = v.w;
          uint4 lo = make_uint4(0, 0, 0, 0);
          if (w && x.lo && row < x.Lq && d < x.D)
            lo = *reinterpret_cast<const uint4*>(x.lo + (o - static_cast<const __nv_bfloat16*>(x.o)) + d);
          const uint32_t ow[4] = {u.x, u.y, u.z, u.w}, lw[4] = {lo.x, lo.y, lo.z, lo.w};
          auto both = [](uint32_t t) {
            return make_float2(__uint_as_float(t << 16), __uint_as_float(t & 0xffff0000u));
          };
#pragma unroll
          for (int e = 0; e < 4; ++e) dot = fma2(both(r[4 * i + e]), add2(both(ow[e]), both(lw[e])), dot);
        }
        tmem_st16((w ? t_do : t_q) + lanes + half * (DP / 4) + c / 2, r);
      }
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(blk.own);
      if (w) s_delta[half][tid & 127] = dot.x + dot.y;
      asm volatile("bar.sync 1, 512;" ::: "memory");
    }
    const float nl = row < x.Lq ? -x.lse2[at] : -INFINITY;
    const float delta = s_delta[0][tid & 127] + s_delta[1][tid & 127];
    if (w && half == 0 && row < x.Lq) x.delta[at] = delta;  // for dk and dv
    const float2 cc = make_float2(c2, c2), ll = make_float2(nl, nl), dd = make_float2(-delta, -delta);
    bool ok = true;
    for (int j = w; j < tiles; j += 2) {
      const uint4 bits = key_bits(p, b, nk, j * kB & ~127);
      const uint32_t word = j & 1 ? (half ? bits.w : bits.z) : (half ? bits.y : bits.x);
      if (!(ok = wait_all(&blk.sd_full[w], j >> 1))) break;
      tc_fence_after();
      if (!idle) {
        float s[32], g[32];
        tmem_ld32_nowait(tS + half * 32, s);
        tmem_ld32_nowait(tS + 64 + half * 32, g);
        tmem_wait_ld();
        tmem_pin<32>(s);
        tmem_pin<32>(g);
        uint32_t r[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float2 e = fma2(make_float2(s[2 * i], s[2 * i + 1]), cc, ll);
          e.x = ex2(e.x), e.y = ex2(e.y);
          e = mul2(e, add2(make_float2(g[2 * i], g[2 * i + 1]), dd));
          s[2 * i] = e.x, s[2 * i + 1] = e.y;
        }
        if (word != 0xffffffffu) {
#pragma unroll
          for (int i = 0; i < 32; ++i) s[i] = word >> i & 1u ? s[i] : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) r[i] = pack_bf16(s[2 * i], s[2 * i + 1]);
        tmem_st16(tS + half * 32, r);  // over scores of this thread's own
        tmem_wait_st();
      }
      tc_fence_before();
      mbar_arrive(&blk.ds_full[w]);
    }
    if (ok && tiles > 0) wait_all(blk.done, 0);
    tc_fence_after();
    if (!idle)
      store_acc<DP / 4>(acc + lanes, static_cast<__nv_bfloat16*>(x.dq) + ((b * x.Lq + row) * x.H + h) * (int64_t)x.D,
                        row < x.Lq, tiles == 0, (2 * w + half) * (DP / 4), x.D, x.scale);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (s_abort) {  // the same for all: nothing writes it after the barrier
    if (warp == kMmaWarp) drain_umma(blk.drain);
    if (warp == kTmaWarp && lane == 0 && tiles > 0) {
      drain_copies(blk.full, issued, Sh::kStages);
    }
    __syncthreads();
  }
  if (warp == kMmaWarp) free_tmem(tmem);
}

template <int DP>
__global__ void __launch_bounds__(BwdShape<DP>::kDkvThreads, 1)
    tc_dkv_kernel(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
                  const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mdo,
                  const __grid_constant__ TcParams p) {
  using Sh = BwdShape<DP>;
  extern __shared__ unsigned char smem_raw[];
  __shared__ uint32_t s_tmem;
  __shared__ volatile int s_abort;
  __shared__ float4 s_stat[2][2][2][kB / 4];  // warpgroup, slot, (-lse2, -delta)
  const Block<DP, true> blk(smem_raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  constexpr int kTmaWarp = 8, kMmaWarp = 9;
  if (warp == kMmaWarp) alloc_tmem(&s_tmem);
  if (tid == 0) {
    s_abort = 0;
    blk.init(128);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_wait();
  pdl_trigger();
  const uint32_t tmem = s_tmem, acc_v = tmem + 256, acc_k = acc_v + DP;
  const Params& x = p.x;
  const int ktiles = (x.Lk + kTile - 1) / kTile, qtiles = (x.Lq + kB - 1) / kB, G = x.H / x.Hkv;
  const int k0 = (int)(blockIdx.x % ktiles) * kTile;
  const int hk = (int)(blockIdx.x / ktiles % x.Hkv);
  const int64_t b = blockIdx.x / ktiles / x.Hkv;
  const int nk = key_count(x, b);
  const int tiles = k0 < nk ? qtiles * G : 0;  // tile i: query head hk * G + i / qtiles, rows (i % qtiles) * 64 ...
  auto wait = [&](uint64_t* bar, uint32_t parity) { return mbar_wait_or(bar, parity & 1, &s_abort, x.err); };
  // the whole warp goes on or gives up together
  auto wait_all = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)) != 0; };

  int issued = 0;  // streamed tiles asked for (lane 0 of the TMA warp)
  if (warp == kTmaWarp) {
    if (lane == 0 && tiles > 0) {
      mbar_expect_tx(blk.own, 2 * Sh::kOpA);
      for (int kb = 0; kb < DP / 64; ++kb) {
        tma_load_4d(blk.a0 + kb * Sh::kBlockA, &mk, kb * 64, k0, hk, (int)b, blk.own);
        tma_load_4d(blk.a1 + kb * Sh::kBlockA, &mv, kb * 64, k0, hk, (int)b, blk.own);
      }
      for (int i = 0; i < tiles; ++i) {
        const int s = i % Sh::kStages, h = hk * G + i / qtiles, r0 = i % qtiles * kB;
        if (!wait(&blk.empty[s], i / Sh::kStages ^ 1)) break;
        mbar_expect_tx(&blk.full[s], 2 * Sh::kOpB);
        for (int kb = 0; kb < DP / 64; ++kb) {
          tma_load_4d(blk.b0 + s * Sh::kOpB + kb * Sh::kBlockB, &mq, kb * 64, r0, h, (int)b, &blk.full[s]);
          tma_load_4d(blk.b1 + s * Sh::kOpB + kb * Sh::kBlockB, &mdo, kb * 64, r0, h, (int)b, &blk.full[s]);
        }
        issued = i + 1;
      }
    }
  } else if (warp == kMmaWarp) {
    const auto is = blk.issue(x.D);
    auto start = [&](int i) {
      const int s = i % Sh::kStages;
      if (!wait_all(&blk.full[s], i / Sh::kStages)) return false;
      tc_fence_after();
      blk.products(is, tmem, i & 1, s);
      return true;
    };
    bool ok = tiles > 0 && wait_all(blk.own, 0) && start(0) && (tiles < 2 || start(1));
    for (int i = 0; i < tiles && ok; ++i) {
      if (!(ok = wait_all(&blk.ds_full[i & 1], i >> 1))) break;
      tc_fence_after();
      const int s = i % Sh::kStages;
      blk.template accumulate<16>(is, acc_v, tmem + (i & 1) * 128, is.t1, s, i == 0);
      blk.template accumulate<16>(is, acc_k, tmem + (i & 1) * 128 + 64, is.t0, s, i == 0);
      umma_done(is.one, &blk.empty[s]);
      if (i == tiles - 1) umma_done(is.one, blk.done);
      if (i + 2 < tiles) ok = start(i + 2);
    }
  } else {
    const int w = warp >> 2, t = tid & 127;
    const int key = k0 + t;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + lanes + w * 128;
    const float c2 = x.scale * kLog2e;
    const float2 cc = make_float2(c2, c2);
    const bool allowed = key < x.Lk && key_ok(x, b, nk, key);
    auto stat = [&](int i) {  // this thread's share of tile i's row statistics
      const int r = i % qtiles * kB + (t & 63);
      const int64_t at = (b * x.H + hk * G + i / qtiles) * x.Lq + r;
      if (t < 64) return i < tiles && r < x.Lq ? -x.lse2[at] : -INFINITY;
      return i < tiles && r < x.Lq ? -x.delta[at] : 0.0f;
    };
    float next = stat(w);
    bool ok = true;
    for (int i = w; i < tiles; i += 2) {
      float4* st = s_stat[w][i >> 1 & 1][0];
      reinterpret_cast<float*>(st)[t] = next;
      asm volatile("bar.sync %0, 128;" ::"r"(1 + w) : "memory");
      next = stat(i + 2);
      if (ok) ok = wait_all(&blk.sd_full[w], i >> 1);
      if (!ok) continue;  // given up: the others still meet at the barrier
      tc_fence_after();
      float s[2][32], g[2][32];
      tmem_ld32_nowait(tS, s[0]);
      tmem_ld32_nowait(tS + 64, g[0]);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        tmem_wait_ld();
        tmem_pin<32>(s[c]);
        tmem_pin<32>(g[c]);
        if (c == 0) {
          tmem_ld32_nowait(tS + 32, s[1]);
          tmem_ld32_nowait(tS + 96, g[1]);
        }
        uint32_t pw[16], dw[16];
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          const float4 l = st[c * 8 + q], d = st[kB / 4 + c * 8 + q];
          float2 e0 = fma2(make_float2(s[c][4 * q], s[c][4 * q + 1]), cc, make_float2(l.x, l.y));
          float2 e1 = fma2(make_float2(s[c][4 * q + 2], s[c][4 * q + 3]), cc, make_float2(l.z, l.w));
          e0.x = ex2(e0.x), e0.y = ex2(e0.y), e1.x = ex2(e1.x), e1.y = ex2(e1.y);
          const float2 d0 = mul2(e0, add2(make_float2(g[c][4 * q], g[c][4 * q + 1]), make_float2(d.x, d.y)));
          const float2 d1 = mul2(e1, add2(make_float2(g[c][4 * q + 2], g[c][4 * q + 3]), make_float2(d.z, d.w)));
          pw[2 * q] = allowed ? pack_bf16(e0.x, e0.y) : 0u, pw[2 * q + 1] = allowed ? pack_bf16(e1.x, e1.y) : 0u;
          dw[2 * q] = allowed ? pack_bf16(d0.x, d0.y) : 0u, dw[2 * q + 1] = allowed ? pack_bf16(d1.x, d1.y) : 0u;
        }
        tmem_st16(tS + c * 16, pw);
        tmem_st16(tS + 64 + c * 16, dw);
      }
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&blk.ds_full[w]);
    }
    if (ok && tiles > 0) wait_all(blk.done, 0);
    tc_fence_after();
    const int64_t at = ((b * x.Lk + key) * x.Hkv + hk) * (int64_t)x.D;
    store_acc<DP>((w ? acc_k : acc_v) + lanes, static_cast<__nv_bfloat16*>(w ? x.dk : x.dv) + at, key < x.Lk,
                  tiles == 0, 0, x.D, w ? x.scale : 1.0f);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (s_abort) {  // the same for all: nothing writes it after the barrier
    if (warp == kMmaWarp) drain_umma(blk.drain);
    if (warp == kTmaWarp && lane == 0 && tiles > 0) {
      mbar_wait(blk.own, 0);
      drain_copies(blk.full, issued, Sh::kStages);
    }
    __syncthreads();
  }
  if (warp == kMmaWarp) free_tmem(tmem);
}

// ---- host ----------------------------------------------------------------------------------
template <int DP>
static int launch_bwd(TcParams& t, cudaStream_t st) {
  using Sh = BwdShape<DP>;
  const Params& x = t.x;
  // before the maps: encoding one needs the device's context, which these calls make current in a new thread
  auto fq = tc_dq_kernel<DP>;
  auto fk = tc_dkv_kernel<DP>;
  if (!set_smem_limit(reinterpret_cast<const void*>(fq), Sh::kDqBytes) ||
      !set_smem_limit(reinterpret_cast<const void*>(fk), Sh::kDkvBytes))
    return HCLSM_ERR_LAUNCH;
  CUtensorMap q64, g64, k128, k64, v128, v64;
  if (!make_map(&q64, x.q, x.D, x.Lq, x.H, x.B, kB) || !make_map(&g64, x.dout, x.D, x.Lq, x.H, x.B, kB) ||
      !make_map(&k128, x.k, x.D, x.Lk, x.Hkv, x.B, kTile) || !make_map(&k64, x.k, x.D, x.Lk, x.Hkv, x.B, kB) ||
      !make_map(&v128, x.v, x.D, x.Lk, x.Hkv, x.B, kTile) || !make_map(&v64, x.v, x.D, x.Lk, x.Hkv, x.B, kB))
    return HCLSM_ERR_UNSUPPORTED;
  t.qtiles = (x.Lq + kTile - 1) / kTile;
  const int64_t gq = (int64_t)t.qtiles * x.H * x.B, gk = (int64_t)((x.Lk + kTile - 1) / kTile) * x.Hkv * x.B;
  if (gq > 0x7fffffff || gk > 0x7fffffff || (int64_t)((x.Lq + kB - 1) / kB) * x.H > 0x7fffffff) return HCLSM_ERR_SHAPE;
  if (const int rc = launch_pdl(fq, (unsigned)gq, Sh::kDqThreads, Sh::kDqBytes, st, k64, v64, t)) return rc;
  return launch_pdl(fk, (unsigned)gk, Sh::kDkvThreads, Sh::kDkvBytes, st, k128, v128, q64, g64, t);
}

// x.delta is room for the row sums; ws: tc_workspace bytes.
int tc_bwd(const Params& p, void* ws, cudaStream_t st) {
  TcParams t = {};
  t.x = p;
  if (const int rc = make_bits(t, ws, st)) return rc;
  return p.D <= 64 ? launch_bwd<64>(t, st) : launch_bwd<128>(t, st);
}

}  // namespace xattn
}  // namespace hclsm
