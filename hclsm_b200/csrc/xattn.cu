// Cross attention: the kernels that serve every type, head size, stride and
// alignment, and the C entry points.
//
// A block keeps TM rows (queries; keys for dk and dv) and walks over tiles of 64 of the
// other side with mma.sync m16n8k16 products; a warp takes 16 rows and half of each
// tile, and the halves are added in order at the end.  An fp32 operand is split
// into three bf16 pieces (8 bits each) when it is staged, one shared-memory plane a
// piece, and the six products of pieces whose order is at most 2 are formed from zero
// and added in fp32: the result is as exact as fp32 arithmetic, at a sixth of the bf16
// rate (170 multiply-adds a clock and SM, 128 on the FP32 pipes) and with a tenth of
// the instructions, which is what counts where few warps are resident.  Rows of planes
// are DP + 8 elements, so that ldmatrix reads every bank once.  One pass over the keys
// with the running maximum and sum of the softmax.  TM 32 where 64 would leave SMs
// without a block.  Forward and backward in fp32, 3 x 333 over 777 ragged, 6 heads over 2
// of 64: 172 us, latency-bound (tensor pipe 24 to 32 % busy, 6 to 8 % of the warps).
#include "xattn.cuh"

namespace hclsm {
namespace xattn {

constexpr int kT = 64;  // rows of a streamed tile
constexpr int kThreads = 256;  // of the row-wise kernel
constexpr int kHalf = kT / 2;  // of it a warp takes
template <int TM> constexpr int kTileThreads = TM * 4;
template <typename T> constexpr int kPieces = sizeof(T) == 4 ? 3 : 1;
template <int DP> constexpr int kLd = DP + 8;

__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, "
      "%2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <bool TRANS>
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], const __nv_bfloat16* p) {
  if constexpr (TRANS)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(smem_u32(p))
                 : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(smem_u32(p))
                 : "memory");
}
// The N leading bf16 pieces of two fp32 values, packed.
template <int N>
__device__ __forceinline__ void pieces(float lo, float hi, uint32_t (&out)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    out[i] = *reinterpret_cast<const uint32_t*>(&h);
    lo -= __uint_as_float(out[i] << 16);
    hi -= __uint_as_float(out[i] & 0xffff0000u);
  }
}

// Rows [r0, r0 + ROWS) of one head as planes of bf16 pieces; rows past n (and, with
// KEYS, keys that are not allowed) and dims past D are zeros.  VEC: D a multiple
// of 4 and aligned rows, four elements a load, all loads in flight first.
template <typename T, int DP, bool KEYS, bool VEC, int ROWS, int NT>
__device__ __forceinline__ void stage(__nv_bfloat16* dst, const View& x, const Params& p, int64_t b, int h, int r0,
                                      int n, const uint8_t* okc) {
  constexpr int N = ROWS * DP / 4 / NT, NP = kPieces<T>, U = N < 8 ? N : 8;
  const T* base = static_cast<const T*>(x.p) + b * x.sb + (int64_t)h * x.sh;
#pragma unroll 1
  for (int i0 = 0; i0 < N; i0 += U) {
    float v[U][4];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int at = threadIdx.x + (i0 + i) * NT, r = at / (DP / 4), d = at % (DP / 4) * 4, row = r0 + r;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[i][e] = 0.0f;
      if (row < n && (!KEYS || okc[r])) {
        const T* src = base + (int64_t)row * x.st + d;
        if constexpr (VEC) {
          if (d < p.D) {
            if constexpr (sizeof(T) == 4) {
              const float4 f = *reinterpret_cast<const float4*>(src);
              v[i][0] = f.x, v[i][1] = f.y, v[i][2] = f.z, v[i][3] = f.w;
            } else {
              const float2 lo = io<T>::ld2(src), hi = io<T>::ld2(src + 2);
              v[i][0] = lo.x, v[i][1] = lo.y, v[i][2] = hi.x, v[i][3] = hi.y;
            }
          }
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (d + e < p.D) v[i][e] = io<T>::ld(src + e);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int at = threadIdx.x + (i0 + i) * NT, r = at / (DP / 4), d = at % (DP / 4) * 4;
      uint32_t lo[NP], hi[NP];
      pieces<NP>(v[i][0], v[i][1], lo);
      pieces<NP>(v[i][2], v[i][3], hi);
#pragma unroll
      for (int k = 0; k < NP; ++k)
        *reinterpret_cast<uint2*>(dst + ((size_t)k * ROWS + r) * kLd<DP> + d) = make_uint2(lo[k], hi[k]);
    }
  }
}

// Four tiles' acc += the products of the pieces a[i] and b[j], order i + j at most NP - 1, smallest first.  b: of two
// pairs of tiles.  The tiles go side by side, because one tile's products wait for each other.
template <int NP>
__device__ __forceinline__ void product4(float (*acc)[4], const uint32_t (&a)[NP][4], const uint32_t (&b)[2][NP][4]) {
  if constexpr (NP == 1) {
#pragma unroll
    for (int t = 0; t < 4; ++t) mma(acc[t], a[0], b[t >> 1][0][2 * (t & 1)], b[t >> 1][0][2 * (t & 1) + 1]);
  } else {
    float part[4][4] = {};
#pragma unroll
    for (int i = NP - 1; i >= 0; --i)
#pragma unroll
      for (int j = NP - 1 - i; j >= 0; --j)
#pragma unroll
        for (int t = 0; t < 4; ++t) mma(part[t], a[i], b[t >> 1][j][2 * (t & 1)], b[t >> 1][j][2 * (t & 1) + 1]);
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[t][e] += part[t][e];
  }
}

// s (the warp's 16 rows x 32) = own rows . streamed rows: a at the warp's first row, b at its first streamed one.
template <int DP, int NP, int ROWS>
__device__ __forceinline__ void dot_tile(float (&s)[4][4], const __nv_bfloat16* a, const __nv_bfloat16* b, int ksteps,
                                         int lane) {
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) s[t][e] = 0.0f;
#pragma unroll 2
  for (int k = 0; k < ksteps; ++k) {
    uint32_t fa[NP][4], fb[2][NP][4];
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      ldmatrix4<false>(fa[i], a + (size_t)i * ROWS * kLd<DP> + (lane & 15) * kLd<DP> + k * 16 + (lane >> 4) * 8);
#pragma unroll
      for (int t = 0; t < 2; ++t)
        ldmatrix4<false>(fb[t][i], b + ((size_t)i * kT + t * 16 + (lane >> 4) * 8 + (lane & 7)) * kLd<DP> + k * 16 +
                                       (lane >> 3 & 1) * 8);
    }
    product4<NP>(s, fa, fb);
  }
}

// acc (16 rows x DP) += w (16 x 32, as dot_tile leaves its products) x the streamed rows at x.
template <int DP, int NP>
__device__ __forceinline__ void gather_tile(float (&acc)[DP / 8][4], const float (&w)[4][4], const __nv_bfloat16* x,
                                            int lane) {
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    uint32_t fa[NP][4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      uint32_t t[NP];
      pieces<NP>(w[2 * u + (e >> 1)][2 * (e & 1)], w[2 * u + (e >> 1)][2 * (e & 1) + 1], t);
#pragma unroll
      for (int i = 0; i < NP; ++i) fa[i][e] = t[i];
    }
#pragma unroll
    for (int j = 0; j < DP / 8; j += 4) {
      uint32_t fb[2][NP][4];
#pragma unroll
      for (int i = 0; i < NP; ++i)
#pragma unroll
        for (int t = 0; t < 2; ++t)
          ldmatrix4<true>(fb[t][i], x + ((size_t)i * kT + u * 16 + (lane & 15)) * kLd<DP> + j * 8 + t * 16 +
                                        (lane >> 4) * 8);
      product4<NP>(acc + j, fa, fb);
    }
  }
}

// The second half's accumulator rows through shared memory (fp32 [rows][DP]): put, then the first half's warps add.
template <int DP>
__device__ __forceinline__ void put_rows(float* dst, const float (&acc)[DP / 8][4], int lane) {
#pragma unroll
  for (int j = 0; j < DP / 8; ++j)
#pragma unroll
    for (int r = 0; r < 2; ++r)
      *reinterpret_cast<float2*>(dst + ((lane >> 2) + 8 * r) * DP + j * 8 + 2 * (lane & 3)) =
          make_float2(acc[j][2 * r], acc[j][2 * r + 1]);
}
// acc = acc * f[row] + src * g[row]
template <int DP>
__device__ __forceinline__ void join_rows(float (&acc)[DP / 8][4], const float* src, const float (&f)[2],
                                          const float (&g)[2], int lane) {
#pragma unroll
  for (int j = 0; j < DP / 8; ++j)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const float2 v =
          *reinterpret_cast<const float2*>(src + ((lane >> 2) + 8 * r) * DP + j * 8 + 2 * (lane & 3));
      acc[j][2 * r] = acc[j][2 * r] * f[r] + v.x * g[r];
      acc[j][2 * r + 1] = acc[j][2 * r + 1] * f[r] + v.y * g[r];
    }
}

template <typename T, int DP>
__device__ __forceinline__ void store_rows(void* dst, const float (&acc)[DP / 8][4], float f, const Params& p,
                                           int64_t b, int L, int H, int h, int r0, int lane,
                                           __nv_bfloat16* lo = nullptr) {
  const int g = lane >> 2, c = lane & 3;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int row = r0 + g + 8 * r;
    if (row >= L) continue;
    T* out = static_cast<T*>(dst) + ((b * L + row) * H + h) * (int64_t)p.D;
#pragma unroll
    for (int j = 0; j < DP / 8; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int d = j * 8 + 2 * c + e;
        if (d < p.D) {
          io<T>::st(out + d, acc[j][2 * r + e] * f);
          if (sizeof(T) == 2 && lo)
            lo[out - static_cast<T*>(dst) + d] = __float2bfloat16_rn(rounding(acc[j][2 * r + e] * f));
        }
      }
  }
}

// Shared memory of a block: NA operands of TM rows and two of 64.
template <typename T, int DP, int TM, int NA> constexpr size_t smem_bytes() {
  const size_t planes = (size_t)kPieces<T> * (NA * TM + 2 * kT) * kLd<DP> * sizeof(__nv_bfloat16);
  const size_t halves = (size_t)NA * TM * DP * sizeof(float);
  return planes > halves ? planes : halves;
}

template <typename T, int DP, bool VEC, int TM>
__global__ void __launch_bounds__(kTileThreads<TM>) fwd_kernel(const __grid_constant__ Params p) {
  constexpr int NT = kTileThreads<TM>, NP = kPieces<T>;
  extern __shared__ uint4 smem4[];
  __nv_bfloat16* sq = reinterpret_cast<__nv_bfloat16*>(smem4);
  __nv_bfloat16* sk = sq + (size_t)NP * TM * kLd<DP>;
  __nv_bfloat16* sv = sk + (size_t)NP * kT * kLd<DP>;
  __shared__ uint8_t okc[kT];
  __shared__ float s_m[TM], s_l[TM];
  const int lane = threadIdx.x & 31, c = lane & 3, g = lane >> 2;
  const int rw = (threadIdx.x >> 5) % (TM / 16) * 16, half = (threadIdx.x >> 5) / (TM / 16);  // the warp's rows, keys
  pdl_wait();
  pdl_trigger();
  const int tiles = (p.Lq + TM - 1) / TM;
  const int r0 = (int)(blockIdx.x % tiles) * TM;
  const int h = (int)(blockIdx.x / tiles % p.H);
  const int64_t b = blockIdx.x / tiles / p.H;
  const int hk = h / (p.H / p.Hkv);
  const int nk = key_count(p, b), ksteps = (p.D + 15) / 16;
  const float c2 = p.scale * kLog2e;
  stage<T, DP, false, VEC, TM, NT>(sq, p.q, p, b, h, r0, p.Lq, nullptr);
  float acc[DP / 8][4] = {}, m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
  for (int k0 = 0; k0 < nk; k0 += kT) {
    __syncthreads();
    for (int i = threadIdx.x; i < kT; i += NT) okc[i] = key_ok(p, b, nk, k0 + i);
    __syncthreads();
    stage<T, DP, true, VEC, kT, NT>(sk, p.k, p, b, hk, k0, nk, okc);
    stage<T, DP, true, VEC, kT, NT>(sv, p.v, p, b, hk, k0, nk, okc);
    __syncthreads();
    float s[4][4];
    dot_tile<DP, NP, TM>(s, sq + rw * kLd<DP>, sk + half * kHalf * kLd<DP>, ksteps, lane);
    float mx[2] = {m[0], m[1]};
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[t][e] = okc[half * kHalf + t * 8 + 2 * c + (e & 1)] ? s[t][e] * c2 : -INFINITY;
        mx[e >> 1] = fmaxf(mx[e >> 1], s[t][e]);
      }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
      mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
      const float base = mx[r] == -INFINITY ? 0.0f : mx[r];  // no allowed key yet: every weight 0
      const float f = ex2(m[r] - base);
      m[r] = mx[r];
      l[r] *= f;
#pragma unroll
      for (int j = 0; j < DP / 8; ++j) acc[j][2 * r] *= f, acc[j][2 * r + 1] *= f;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          s[t][2 * r + e] = ex2(s[t][2 * r + e] - base);
          l[r] += s[t][2 * r + e];
        }
    }
    gather_tile<DP, NP>(acc, s, sv + half * kHalf * kLd<DP>, lane);
  }
  __syncthreads();  // the tiles are done with
  float* other = reinterpret_cast<float*>(smem4) + (size_t)rw * DP;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    if (half && c == 0) s_m[rw + g + 8 * r] = m[r], s_l[rw + g + 8 * r] = l[r];
  }
  if (half) put_rows<DP>(other, acc, lane);
  __syncthreads();
  if (half) return;
  float f0[2], f1[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const float m1 = s_m[rw + g + 8 * r], l1 = s_l[rw + g + 8 * r], mx = fmaxf(m[r], m1);
    // a half without a maximum holds zeros, or NaN that has to stay
    f0[r] = m[r] == -INFINITY ? 1.0f : ex2(m[r] - mx);
    f1[r] = m1 == -INFINITY ? 1.0f : ex2(m1 - mx);
    const float sum = l[r] * f0[r] + l1 * f1[r];
    const bool empty = sum == 0.0f;  // a row with a key sums to at least 1
    const float inv = empty ? 0.0f : 1.0f / sum;
    f0[r] *= inv, f1[r] *= inv;
    const int row = r0 + rw + g + 8 * r;
    if (p.lse2 && c == 0 && row < p.Lq) p.lse2[(b * p.H + h) * p.Lq + row] = empty ? INFINITY : mx + log2f(sum);
  }
  join_rows<DP>(acc, other, f0, f1, lane);
  store_rows<T, DP>(p.o, acc, 1.0f, p, b, p.Lq, p.H, h, r0 + rw, lane, p.lo);
}

// dq (KEYROWS false): rows are queries, columns keys, acc += ds k.
// dk, dv (KEYROWS): rows are keys, columns queries, so the scores are formed transposed;
// acc (dk) += ds^T q and acc2 (dv) += p^T do, over the query heads that share the key head one after another, or
// (p.part) over one of them, whose sums join_heads_kernel adds.
template <typename T, int DP, bool VEC, int TM, bool KEYROWS>
__global__ void __launch_bounds__(kTileThreads<TM>) bwd_kernel(const __grid_constant__ Params p) {
  constexpr int NT = kTileThreads<TM>, NP = kPieces<T>;
  extern __shared__ uint4 smem4[];
  __nv_bfloat16* a0 = reinterpret_cast<__nv_bfloat16*>(smem4);  // q, do or k, v
  __nv_bfloat16* a1 = a0 + (size_t)NP * TM * kLd<DP>;
  __nv_bfloat16* b0 = a1 + (size_t)NP * TM * kLd<DP>;           // k, v or q, do
  __nv_bfloat16* b1 = b0 + (size_t)NP * kT * kLd<DP>;
  __shared__ uint8_t okc[kT];                  // of the keys
  __shared__ float s_lse[kT], s_delta[kT];     // of the queries
  constexpr int KROWS = KEYROWS ? TM : kT, QROWS = KEYROWS ? kT : TM;
  const int lane = threadIdx.x & 31, c = lane & 3, g = lane >> 2;
  const int rw = (threadIdx.x >> 5) % (TM / 16) * 16, half = (threadIdx.x >> 5) / (TM / 16);
  pdl_wait();
  pdl_trigger();
  const int own = KEYROWS ? p.Lk : p.Lq, heads = KEYROWS ? p.Hkv : p.H, G = p.H / p.Hkv;
  const int tiles = (own + TM - 1) / TM;
  const bool apart = KEYROWS && p.part;
  const int only = apart ? (int)(blockIdx.x % G) : 0;  // the query head of this block
  const unsigned int block = apart ? blockIdx.x / G : blockIdx.x;
  const int r0 = (int)(block % tiles) * TM;
  const int h = (int)(block / tiles % heads);
  const int64_t b = block / tiles / heads;
  const int nk = key_count(p, b), ksteps = (p.D + 15) / 16;
  const float c2 = p.scale * kLog2e;
  auto keys = [&](__nv_bfloat16* k, __nv_bfloat16* v, int hk, int k0) {
    for (int i = threadIdx.x; i < KROWS; i += NT) okc[i] = key_ok(p, b, nk, k0 + i);
    __syncthreads();
    stage<T, DP, true, VEC, KROWS, NT>(k, p.k, p, b, hk, k0, nk, okc);
    stage<T, DP, true, VEC, KROWS, NT>(v, p.v, p, b, hk, k0, nk, okc);
  };
  auto queries = [&](__nv_bfloat16* q, __nv_bfloat16* d, int hq, int q0) {
    stage<T, DP, false, VEC, QROWS, NT>(q, p.q, p, b, hq, q0, p.Lq, nullptr);
    stage<T, DP, false, VEC, QROWS, NT>(d, p.dout, p, b, hq, q0, p.Lq, nullptr);
    for (int i = threadIdx.x; i < QROWS; i += NT) {  // rows past the end weigh nothing
      const int64_t at = (b * p.H + hq) * p.Lq + q0 + i;
      s_lse[i] = q0 + i < p.Lq ? p.lse2[at] : INFINITY;
      s_delta[i] = q0 + i < p.Lq ? p.delta[at] : 0.0f;
    }
  };
  float acc[DP / 8][4] = {}, acc2[KEYROWS ? DP / 8 : 1][4] = {};
  const int n = KEYROWS ? p.Lq : nk;  // streamed rows of a head
  const int loops = KEYROWS ? (r0 < nk ? (apart ? 1 : G) : 0) : 1;
  if (loops > 0) {
    if constexpr (KEYROWS) keys(a0, a1, h, r0);
    else queries(a0, a1, h, r0);
  }
  for (int q = 0; q < loops; ++q)
    for (int s0 = 0; s0 < n; s0 += kT) {
      __syncthreads();
      if constexpr (KEYROWS) queries(b0, b1, h * G + only + q, s0);
      else keys(b0, b1, h / G, s0);
      __syncthreads();
      float s[4][4], d[4][4];
      const int at = half * kHalf * kLd<DP>;
      dot_tile<DP, NP, TM>(s, a0 + rw * kLd<DP>, b0 + at, ksteps, lane);
      dot_tile<DP, NP, TM>(d, a1 + rw * kLd<DP>, b1 + at, ksteps, lane);
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int row = rw + g + 8 * (e >> 1), col = half * kHalf + t * 8 + 2 * c + (e & 1);
          const int key = KEYROWS ? row : col, query = KEYROWS ? col : row;
          s[t][e] = okc[key] ? ex2(s[t][e] * c2 - s_lse[query]) : 0.0f;
          d[t][e] = okc[key] ? s[t][e] * (d[t][e] - s_delta[query]) : 0.0f;
        }
      gather_tile<DP, NP>(acc, d, b0 + at, lane);
      if constexpr (KEYROWS) gather_tile<DP, NP>(acc2, s, b1 + at, lane);
    }
  __syncthreads();  // the tiles are done with
  float* other = reinterpret_cast<float*>(smem4) + (size_t)rw * DP;
  if (half) {
    put_rows<DP>(other, acc, lane);
    if constexpr (KEYROWS) put_rows<DP>(other + TM * DP, acc2, lane);
  }
  __syncthreads();
  if (half) return;
  const float one[2] = {1.0f, 1.0f};
  join_rows<DP>(acc, other, one, one, lane);
  if constexpr (KEYROWS) {
    join_rows<DP>(acc2, other + TM * DP, one, one, lane);
    if (apart) {
      const int64_t n = (int64_t)p.B * p.Lk * p.Hkv * p.D;
      store_rows<float, DP>(p.part + only * n, acc, p.scale, p, b, p.Lk, p.Hkv, h, r0 + rw, lane);
      store_rows<float, DP>(p.part + (G + only) * n, acc2, 1.0f, p, b, p.Lk, p.Hkv, h, r0 + rw, lane);
      return;
    }
    store_rows<T, DP>(p.dk, acc, p.scale, p, b, p.Lk, p.Hkv, h, r0 + rw, lane);
    store_rows<T, DP>(p.dv, acc2, 1.0f, p, b, p.Lk, p.Hkv, h, r0 + rw, lane);
  } else {
    store_rows<T, DP>(p.dq, acc, p.scale, p, b, p.Lq, p.H, h, r0 + rw, lane);
  }
}

// dk (blockIdx.y 0) and dv (1) from the query heads' parts, in order.
template <typename T>
__global__ void __launch_bounds__(kThreads) join_heads_kernel(const __grid_constant__ Params p) {
  pdl_wait();
  pdl_trigger();
  const int64_t n = (int64_t)p.B * p.Lk * p.Hkv * p.D, i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (i >= n) return;
  const int G = p.H / p.Hkv;
  const float* part = p.part + blockIdx.y * G * n + i;
  float a = 0.0f;
  for (int g = 0; g < G; ++g) a += part[g * n];
  io<T>::st(static_cast<T*>(blockIdx.y ? p.dv : p.dk) + i, a);
}

// Whether dk and dv take a block a query head: shared key heads, and too few blocks for the SMs otherwise.
bool heads_apart(const Params& p) {
  return p.H > p.Hkv && (int64_t)((p.Lk + 31) / 32) * p.Hkv * p.B < 2 * (int64_t)num_sms();
}
size_t part_bytes(const Params& p) {
  return heads_apart(p) ? (size_t)2 * p.B * p.Lk * p.H * p.D * sizeof(float) : 0;
}

// delta_i = do_i . o_i, one warp a row.
template <typename T>
__global__ void __launch_bounds__(kThreads) delta_kernel(const __grid_constant__ Params p) {
  pdl_wait();
  pdl_trigger();
  const int64_t row = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= (int64_t)p.B * p.Lq * p.H) return;
  const int h = (int)(row % p.H);
  const int64_t bt = row / p.H, b = bt / p.Lq, t = bt % p.Lq;
  const T* o = static_cast<const T*>(p.o) + row * p.D;
  const T* g = static_cast<const T*>(p.dout.p) + b * p.dout.sb + t * p.dout.st + h * p.dout.sh;
  float a = 0.0f;
  for (int d = lane; d < p.D; d += 32) {
    float v = io<T>::ld(o + d);
    if (sizeof(T) == 2 && p.lo) v += __bfloat162float(p.lo[row * p.D + d]);
    a += v * io<T>::ld(g + d);
  }
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) a += __shfl_xor_sync(0xffffffffu, a, s);
  if (lane == 0) p.delta[(b * p.H + h) * p.Lq + t] = a;
}

template <typename T, int DP, bool VEC, int TM>
int launch_rows(const Params& p, int which, cudaStream_t st) {  // 0 forward, 1 dq, 2 dk and dv
  const int64_t rows = which == 2 ? p.Lk : p.Lq, heads = which == 2 ? p.Hkv : p.H;
  const bool apart = which == 2 && p.part;
  const int64_t grid = (rows + TM - 1) / TM * heads * p.B * (apart ? p.H / p.Hkv : 1);
  if (grid > 0x7fffffff) return HCLSM_ERR_SHAPE;
  if (grid == 0) return HCLSM_OK;
  const size_t bytes = which == 0 ? smem_bytes<T, DP, TM, 1>() : smem_bytes<T, DP, TM, 2>();
  auto f = which == 0   ? fwd_kernel<T, DP, VEC, TM>
           : which == 1 ? bwd_kernel<T, DP, VEC, TM, false>
                        : bwd_kernel<T, DP, VEC, TM, true>;
  if (!set_smem_limit(reinterpret_cast<const void*>(f), bytes)) return HCLSM_ERR_LAUNCH;
  const int rc = launch_pdl(f, (unsigned)grid, kTileThreads<TM>, bytes, st, p);
  if (rc || !apart) return rc;
  const int64_t n = (int64_t)p.B * p.Lk * p.Hkv * p.D;
  return launch_pdl(join_heads_kernel<T>, dim3((unsigned)((n + kThreads - 1) / kThreads), 2), kThreads, 0, st, p);
}

template <typename T, int DP, bool VEC>
int run(const Params& p, bool bwd, cudaStream_t st) {
  for (int which = bwd ? 1 : 0; which < (bwd ? 3 : 1); ++which) {
    const int64_t rows = which == 2 ? p.Lk : p.Lq, heads = which == 2 ? p.Hkv : p.H;
    const bool small = (rows + 63) / 64 * heads * p.B < 2 * (int64_t)num_sms();
    const int rc = small ? launch_rows<T, DP, VEC, 32>(p, which, st) : launch_rows<T, DP, VEC, 64>(p, which, st);
    if (rc) return rc;
  }
  return HCLSM_OK;
}

template <typename T>
bool rows4(const View& v) {  // four elements at a time
  const int64_t e = 16 / sizeof(T) / (sizeof(T) == 2 ? 2 : 1);
  return reinterpret_cast<uintptr_t>(v.p) % (e * sizeof(T)) == 0 && v.sb % e == 0 && v.st % e == 0 && v.sh % e == 0;
}
template <typename T, int DP>
int run_any(const Params& p, bool bwd, cudaStream_t st) {
  const bool vec = p.D % 4 == 0 && rows4<T>(p.q) && rows4<T>(p.k) && rows4<T>(p.v) && (!bwd || rows4<T>(p.dout));
  return vec ? run<T, DP, true>(p, bwd, st) : run<T, DP, false>(p, bwd, st);
}
template <typename T>
int dispatch(const Params& p, bool bwd, cudaStream_t st) {
  if (p.D <= 32) return run_any<T, 32>(p, bwd, st);
  if (p.D <= 64) return run_any<T, 64>(p, bwd, st);
  return run_any<T, 128>(p, bwd, st);
}

int launch_delta(const Params& p, int dtype, cudaStream_t st) {
  const int64_t rows = (int64_t)p.B * p.Lq * p.H, grid = (rows + 7) / 8;
  if (grid > 0x7fffffff) return HCLSM_ERR_SHAPE;
  if (grid == 0) return HCLSM_OK;
  return dtype == HCLSM_F32 ? launch_pdl(delta_kernel<float>, (unsigned)grid, kThreads, 0, st, p)
                            : launch_pdl(delta_kernel<__nv_bfloat16>, (unsigned)grid, kThreads, 0, st, p);
}

size_t delta_bytes(const Params& p) { return ((size_t)p.B * p.H * p.Lq * sizeof(float) + 15) / 16 * 16; }

int check(const hclsm_xattn_args* a) {
  if (!a) return HCLSM_ERR_NULL;
  if (a->dtype != HCLSM_F32 && a->dtype != HCLSM_BF16) return HCLSM_ERR_DTYPE;
  if (a->B < 0 || a->Lq < 0 || a->Lk < 0 || a->H < 1 || a->Hkv < 1 || a->H % a->Hkv || a->D < 1 || a->D > 128 ||
      !(a->scale > 0.0f) || a->scale > 3.0e38f)
    return HCLSM_ERR_SHAPE;
  return HCLSM_OK;
}

Params params(const hclsm_xattn_args* a) {
  Params p = {};
  p.q = view(a->q, a->B, a->Lq, a->H), p.dout = view(a->dout, a->B, a->Lq, a->H);
  p.k = view(a->k, a->B, a->Lk, a->Hkv), p.v = view(a->v, a->B, a->Lk, a->Hkv);
  p.o = a->o, p.dq = a->dq, p.dk = a->dk, p.dv = a->dv;
  p.lse2 = a->lse2;
  p.lo = a->dtype == HCLSM_BF16 ? static_cast<__nv_bfloat16*>(a->lo) : nullptr;
  p.lens = a->lens, p.mask = a->mask, p.mask_sb = a->mask_sb;
  p.B = a->B, p.Lq = a->Lq, p.Lk = a->Lk, p.H = a->H, p.Hkv = a->Hkv, p.D = a->D;
  p.scale = a->scale;
  p.err = device_err_ptr();
  return p;
}

}  // namespace xattn
}  // namespace hclsm

using namespace hclsm;

// The split form or the tiles, by the time that each takes on a B200 (us).  The split form: a start, and the keys'
// and values read once for every 16 rows of a key head (bytes a us; more than one reading comes from L2).  The
// tiles: a start, and a time a tile of keys (128 on the tensor cores, 64 otherwise) of each wave of blocks.  Fitted
// to 521 shapes (1 to 64 entries, 1 to 64 heads, 1 to 256 queries over 200 to 16384 keys, heads of 64 and 128, both
// types): picking by it costs 1.7 % over picking the faster one, always the split form for up to 16 rows and never
// else 46 %.  Heads of 32 take the constants of 64 and heads of 96 those of 128, without a fit of their own.
static bool use_split(const xattn::Params& p, int dtype, bool tc) {
  const bool f32 = dtype == HCLSM_F32, small = p.D <= 64;
  const int e = f32 ? 4 : 2;
  auto ok = [&](const xattn::View& v) {
    return reinterpret_cast<uintptr_t>(v.p) % 16 == 0 && v.sb * e % 16 == 0 && v.st * e % 16 == 0 && v.sh * e % 16 == 0;
  };
  if (p.Lk == 0 || p.D % 32 || !ok(p.k) || !ok(p.v)) return false;
  const double rows16 = ((int64_t)p.Lq * (p.H / p.Hkv) + 15) / 16;
  const double bytes = (double)p.B * p.Hkv * rows16 * p.Lk * p.D * 2 * e;
  const double rate = f32 ? (small ? 5.2e6 : 4.3e6) : (rows16 == 1 ? 4.4e6 : 6.5e6);
  const double split = (rows16 == 1 ? (small ? 6.0 : 7.5) : (small ? 8.0 : 11.0)) + bytes / rate;
  double tiles;
  if (tc) {
    const int qt = p.Lq <= 128 ? 1 : 2, resident = num_sms() * (qt == 1 ? 2 : 1);
    const int64_t blocks = (int64_t)((p.Lq + 128 * qt - 1) / (128 * qt)) * p.H * p.B;
    tiles = 4.0 + (double)((blocks + resident - 1) / resident) * ((p.Lk + 127) / 128) * (small ? 1.3 : 1.7);
  } else {
    const double waves = (double)((p.Lq + 31) / 32) * p.H * p.B / num_sms();
    tiles = 4.0 + (waves > 1.0 ? waves : 1.0) * ((p.Lk + 63) / 64) * (small ? 4.0 : 8.5);
  }
  return split < tiles;
}
// Which kernels serve a forward call.
enum Path { kTiles, kTensor, kSplit };
static Path fwd_path(const xattn::Params& p, int dtype) {
  const bool tc = dtype == HCLSM_BF16 && xattn::tc_ok(p, false);
  return use_split(p, dtype, tc) ? kSplit : tc ? kTensor : kTiles;
}

extern "C" size_t hclsm_xattn_fwd_workspace_size(const hclsm_xattn_args* a) {
  if (xattn::check(a)) return 0;
  const xattn::Params p = xattn::params(a);
  const Path path = fwd_path(p, a->dtype);
  return path == kSplit ? xattn::split_workspace(p, a->dtype) : path == kTensor ? xattn::tc_workspace(p) : 0;
}

extern "C" int hclsm_xattn_fwd(const hclsm_xattn_args* a, void* ws, size_t ws_bytes, void* stream) {
  if (const int rc = xattn::check(a)) return rc;
  if ((int64_t)a->B * a->Lq == 0) return HCLSM_OK;
  if (!a->q.p || !a->o || (a->Lk > 0 && (!a->k.p || !a->v.p))) return HCLSM_ERR_NULL;
  if (reinterpret_cast<uintptr_t>(a->lo) % 16) return HCLSM_ERR_ALIGN;
  const xattn::Params p = xattn::params(a);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const Path path = fwd_path(p, a->dtype);
  if (path == kTiles)
    return a->dtype == HCLSM_F32 ? xattn::dispatch<float>(p, false, st) : xattn::dispatch<__nv_bfloat16>(p, false, st);
  const size_t need = path == kSplit ? xattn::split_workspace(p, a->dtype) : xattn::tc_workspace(p);
  if (ws_bytes < need || (need && !ws)) return HCLSM_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(ws) % 16) return HCLSM_ERR_ALIGN;
  return path == kSplit ? xattn::split_fwd(p, a->dtype, ws, st) : xattn::tc_fwd(p, ws, st);
}

static bool use_tc_bwd(const xattn::Params& p, int dtype) {
  auto al = [](const void* q) { return reinterpret_cast<uintptr_t>(q) % 16 == 0; };
  return dtype == HCLSM_BF16 && xattn::tc_ok(p, true) && al(p.dq) && al(p.dk) && al(p.dv);
}

extern "C" size_t hclsm_xattn_bwd_workspace_size(const hclsm_xattn_args* a) {
  if (xattn::check(a)) return 0;
  const xattn::Params p = xattn::params(a);
  return xattn::delta_bytes(p) + (use_tc_bwd(p, a->dtype) ? xattn::tc_workspace(p) : xattn::part_bytes(p));
}

extern "C" int hclsm_xattn_bwd(const hclsm_xattn_args* a, void* ws, size_t ws_bytes, void* stream) {
  if (const int rc = xattn::check(a)) return rc;
  if (a->B == 0) return HCLSM_OK;
  if (a->Lq > 0 && (!a->q.p || !a->o || !a->dout.p || !a->dq || !a->lse2)) return HCLSM_ERR_NULL;
  if (a->Lk > 0 && (!a->k.p || !a->v.p || !a->dk || !a->dv)) return HCLSM_ERR_NULL;
  if (reinterpret_cast<uintptr_t>(a->lo) % 16) return HCLSM_ERR_ALIGN;
  const size_t need = hclsm_xattn_bwd_workspace_size(a);
  if (ws_bytes < need || (need && !ws)) return HCLSM_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(ws) % 16) return HCLSM_ERR_ALIGN;
  xattn::Params p = xattn::params(a);
  p.delta = static_cast<float*>(ws);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  void* more = static_cast<char*>(ws) + xattn::delta_bytes(p);
  if (use_tc_bwd(p, a->dtype)) return xattn::tc_bwd(p, more, st);
  if (xattn::heads_apart(p)) p.part = static_cast<float*>(more);
  if (const int rc = xattn::launch_delta(p, a->dtype, st)) return rc;
  return a->dtype == HCLSM_F32 ? xattn::dispatch<float>(p, true, st) : xattn::dispatch<__nv_bfloat16>(p, true, st);
}
