// Cross attention: the kernels that serve every type, head size, stride and
// alignment (fp32 arithmetic throughout), and the C entry points.
//
// A block keeps TM rows (queries; keys for dk and dv) and walks over tiles of 64 of the
// other side: TM x 64 scores, 4 x 4 a thread; operands are staged in shared memory as
// fp32 rows of DP + 4 floats (the pad keeps the 16 lanes that read different rows on
// different banks).  One pass over the keys with the running maximum and sum of the
// softmax.  Bound: the FP32 pipes.  TM 64 reads the least; TM 32 where 64 would leave
// SMs without a block.
#include "xattn.cuh"

namespace hclsm {
namespace xattn {

constexpr int kT = 64;  // rows of a streamed tile
constexpr int kThreads = 256;  // of the row-wise kernel
template <int TM> constexpr int kTileThreads = TM * 4;

// Rows [r0, r0 + ROWS) of one head as fp32 rows of DP + 4; rows past n (and, with
// KEYS, keys that are not allowed) and dims past D are zeros.  VEC: D a multiple
// of 4 and aligned rows, four elements a load, all loads in flight first.
template <typename T, int DP, bool KEYS, bool VEC, int ROWS, int NT>
__device__ __forceinline__ void stage(float* dst, const View& x, const Params& p, int64_t b, int h, int r0, int n,
                                      const uint8_t* okc) {
  const T* base = static_cast<const T*>(x.p) + b * x.sb + (int64_t)h * x.sh;
  if constexpr (VEC) {
    constexpr int N = ROWS * DP / 4 / NT;
    float4 v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = threadIdx.x + i * NT, r = at / (DP / 4), d = at % (DP / 4) * 4, row = r0 + r;
      v[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (d < p.D && row < n && (!KEYS || okc[r])) {
        const T* src = base + (int64_t)row * x.st + d;
        if constexpr (sizeof(T) == 4) {
          v[i] = *reinterpret_cast<const float4*>(src);
        } else {
          const float2 lo = io<T>::ld2(src), hi = io<T>::ld2(src + 2);
          v[i] = make_float4(lo.x, lo.y, hi.x, hi.y);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = threadIdx.x + i * NT, r = at / (DP / 4), d = at % (DP / 4) * 4;
      *reinterpret_cast<float4*>(dst + r * (DP + 4) + d) = v[i];
    }
  } else {
    for (int i = threadIdx.x; i < ROWS * DP; i += NT) {
      const int r = i / DP, d = i % DP, row = r0 + r;
      const bool ok = d < p.D && row < n && (!KEYS || okc[r]);
      dst[r * (DP + 4) + d] = ok ? io<T>::ld(base + (int64_t)row * x.st + d) : 0.0f;
    }
  }
}

// acc[i][j] += sum_d a[4 ty + i][d] * b[tx + 16 j][d]
template <int DP>
__device__ __forceinline__ void dot_tile(float (&acc)[4][4], const float* a, const float* b, int ty, int tx) {
#pragma unroll 4
  for (int d = 0; d < DP; d += 4) {
    float4 x[4], y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = *reinterpret_cast<const float4*>(a + (4 * ty + i) * (DP + 4) + d);
      y[i] = *reinterpret_cast<const float4*>(b + (tx + 16 * i) * (DP + 4) + d);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        acc[i][j] = fmaf(x[i].x, y[j].x, acc[i][j]);
        acc[i][j] = fmaf(x[i].y, y[j].y, acc[i][j]);
        acc[i][j] = fmaf(x[i].z, y[j].z, acc[i][j]);
        acc[i][j] = fmaf(x[i].w, y[j].w, acc[i][j]);
      }
  }
}

// Dims of a thread: 4 tx ... + 3 of each 64, or 2 tx, + 1 of 32.
template <int DP> constexpr int kRun = DP == 32 ? 2 : 4;
template <int DP>
__device__ __forceinline__ int dim_of(int n, int tx) {
  return n / kRun<DP> * 16 * kRun<DP> + tx * kRun<DP> + n % kRun<DP>;
}

// out[i][n] += sum_c w[4 ty + i][c] * x[c][dim_of(n)]
template <int DP>
__device__ __forceinline__ void gather_tile(float (&out)[4][DP / 16], const float* w, const float* x, int ty, int tx) {
#pragma unroll 2
  for (int c = 0; c < kT; c += 4) {
    float a[4][4];  // [row][c]
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 v = *reinterpret_cast<const float4*>(w + (4 * ty + i) * (kT + 4) + c);
      a[i][0] = v.x, a[i][1] = v.y, a[i][2] = v.z, a[i][3] = v.w;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int n = 0; n < DP / 16; n += kRun<DP>) {
        float y[kRun<DP>];
        const float* src = x + (c + k) * (DP + 4) + dim_of<DP>(n, tx);
        if constexpr (kRun<DP> == 4) {
          const float4 v = *reinterpret_cast<const float4*>(src);
          y[0] = v.x, y[1] = v.y, y[2] = v.z, y[3] = v.w;
        } else {
          const float2 v = *reinterpret_cast<const float2*>(src);
          y[0] = v.x, y[1] = v.y;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < kRun<DP>; ++e) out[i][n + e] = fmaf(a[i][k], y[e], out[i][n + e]);
      }
  }
}

template <typename T, int DP>
__device__ __forceinline__ void store_rows(void* dst, const float (&acc)[4][DP / 16], const float (&f)[4],
                                           const Params& p, int64_t b, int L, int H, int h, int r0, int ty, int tx) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = r0 + 4 * ty + i;
    if (row >= L) continue;
    T* out = static_cast<T*>(dst) + ((b * L + row) * H + h) * (int64_t)p.D;
#pragma unroll
    for (int n = 0; n < DP / 16; ++n) {
      const int d = dim_of<DP>(n, tx);
      if (d < p.D) io<T>::st(out + d, acc[i][n] * f[i]);
    }
  }
}

template <int DP> constexpr size_t row_floats = DP + 4;

// Shared memory of a block: NA operands of TM rows, NB of 64, NS score tiles.
template <int DP, int TM, int NA, int NB, int NS> constexpr size_t smem_bytes() {
  return 4 * ((NA * TM + NB * kT) * row_floats<DP> + (size_t)NS * TM * (kT + 4));
}

template <typename T, int DP, bool VEC, int TM>
__global__ void __launch_bounds__(kTileThreads<TM>) fwd_kernel(const __grid_constant__ Params p) {
  constexpr int NT = kTileThreads<TM>;
  extern __shared__ float4 smem4[];
  float* sq = reinterpret_cast<float*>(smem4);
  float* sk = sq + TM * row_floats<DP>;
  float* sv = sk + kT * row_floats<DP>;
  float* sp = sv + kT * row_floats<DP>;
  __shared__ uint8_t okc[kT];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  pdl_wait();
  pdl_trigger();
  const int tiles = (p.Lq + TM - 1) / TM;
  const int r0 = (int)(blockIdx.x % tiles) * TM;
  const int h = (int)(blockIdx.x / tiles % p.H);
  const int64_t b = blockIdx.x / tiles / p.H;
  const int hk = h / (p.H / p.Hkv);
  const int nk = key_count(p, b);
  const float c2 = p.scale * kLog2e;
  stage<T, DP, false, VEC, TM, NT>(sq, p.q, p, b, h, r0, p.Lq, nullptr);
  float acc[4][DP / 16] = {}, m[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) m[i] = -INFINITY, l[i] = 0.0f;
  for (int k0 = 0; k0 < nk; k0 += kT) {
    __syncthreads();
    if (threadIdx.x < kT) okc[threadIdx.x] = key_ok(p, b, nk, k0 + threadIdx.x);
    __syncthreads();
    stage<T, DP, true, VEC, kT, NT>(sk, p.k, p, b, hk, k0, nk, okc);
    stage<T, DP, true, VEC, kT, NT>(sv, p.v, p, b, hk, k0, nk, okc);
    __syncthreads();
    float s[4][4] = {};
    dot_tile<DP>(s, sq, sk, ty, tx);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float mx = m[i];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[i][j] = okc[tx + 16 * j] ? s[i][j] * c2 : -INFINITY;
        mx = fmaxf(mx, s[i][j]);
      }
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      const float base = mx == -INFINITY ? 0.0f : mx;  // no allowed key yet: every weight 0
      const float f = exp2f(m[i] - base);
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float e = exp2f(s[i][j] - base);
        sp[(4 * ty + i) * (kT + 4) + tx + 16 * j] = e;
        sum += e;
      }
      m[i] = mx;
      l[i] = l[i] * f + sum;
#pragma unroll
      for (int n = 0; n < DP / 16; ++n) acc[i][n] *= f;
    }
    __syncwarp();  // a warp's rows of weights are its own
    gather_tile<DP>(acc, sp, sv, ty, tx);
  }
  float inv[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], o);
    const bool empty = l[i] == 0.0f;  // a row with a key sums to at least 1
    inv[i] = empty ? 0.0f : 1.0f / l[i];
    const int row = r0 + 4 * ty + i;
    if (p.lse2 && tx == 0 && row < p.Lq) p.lse2[(b * p.H + h) * p.Lq + row] = empty ? INFINITY : m[i] + log2f(l[i]);
  }
  store_rows<T, DP>(p.o, acc, inv, p, b, p.Lq, p.H, h, r0, ty, tx);
}

template <typename T, int DP, bool VEC, int TM>
__global__ void __launch_bounds__(kTileThreads<TM>) dq_kernel(const __grid_constant__ Params p) {
  constexpr int NT = kTileThreads<TM>;
  extern __shared__ float4 smem4[];
  float* sq = reinterpret_cast<float*>(smem4);
  float* sdo = sq + TM * row_floats<DP>;
  float* sk = sdo + TM * row_floats<DP>;
  float* sv = sk + kT * row_floats<DP>;
  float* sds = sv + kT * row_floats<DP>;
  __shared__ uint8_t okc[kT];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  pdl_wait();
  pdl_trigger();
  const int tiles = (p.Lq + TM - 1) / TM;
  const int r0 = (int)(blockIdx.x % tiles) * TM;
  const int h = (int)(blockIdx.x / tiles % p.H);
  const int64_t b = blockIdx.x / tiles / p.H;
  const int hk = h / (p.H / p.Hkv);
  const int nk = key_count(p, b);
  const float c2 = p.scale * kLog2e;
  stage<T, DP, false, VEC, TM, NT>(sq, p.q, p, b, h, r0, p.Lq, nullptr);
  stage<T, DP, false, VEC, TM, NT>(sdo, p.dout, p, b, h, r0, p.Lq, nullptr);
  float acc[4][DP / 16] = {}, lse[4], delta[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {  // rows past the end weigh nothing
    const int row = r0 + 4 * ty + i;
    const int64_t at = (b * p.H + h) * p.Lq + row;
    lse[i] = row < p.Lq ? p.lse2[at] : INFINITY;
    delta[i] = row < p.Lq ? p.delta[at] : 0.0f;
  }
  for (int k0 = 0; k0 < nk; k0 += kT) {
    __syncthreads();
    if (threadIdx.x < kT) okc[threadIdx.x] = key_ok(p, b, nk, k0 + threadIdx.x);
    __syncthreads();
    stage<T, DP, true, VEC, kT, NT>(sk, p.k, p, b, hk, k0, nk, okc);
    stage<T, DP, true, VEC, kT, NT>(sv, p.v, p, b, hk, k0, nk, okc);
    __syncthreads();
    float s[4][4] = {}, dp[4][4] = {};
    dot_tile<DP>(s, sq, sk, ty, tx);
    dot_tile<DP>(dp, sdo, sv, ty, tx);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float w = okc[tx + 16 * j] ? exp2f(s[i][j] * c2 - lse[i]) : 0.0f;
        sds[(4 * ty + i) * (kT + 4) + tx + 16 * j] = w * (dp[i][j] - delta[i]);
      }
    __syncwarp();
    gather_tile<DP>(acc, sds, sk, ty, tx);
  }
  const float f[4] = {p.scale, p.scale, p.scale, p.scale};
  store_rows<T, DP>(p.dq, acc, f, p, b, p.Lq, p.H, h, r0, ty, tx);
}

// Rows are keys, columns queries: the scores are formed transposed.
template <typename T, int DP, bool VEC, int TM>
__global__ void __launch_bounds__(kTileThreads<TM>) dkv_kernel(const __grid_constant__ Params p) {
  constexpr int NT = kTileThreads<TM>;
  extern __shared__ float4 smem4[];
  float* sk = reinterpret_cast<float*>(smem4);
  float* sv = sk + TM * row_floats<DP>;
  float* sq = sv + TM * row_floats<DP>;
  float* sdo = sq + kT * row_floats<DP>;
  float* sp = sdo + kT * row_floats<DP>;
  float* sds = sp + TM * (kT + 4);
  __shared__ uint8_t okc[TM];
  __shared__ float s_lse[kT], s_delta[kT];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  pdl_wait();
  pdl_trigger();
  const int tiles = (p.Lk + TM - 1) / TM;
  const int k0 = (int)(blockIdx.x % tiles) * TM;
  const int hk = (int)(blockIdx.x / tiles % p.Hkv);
  const int64_t b = blockIdx.x / tiles / p.Hkv;
  const int G = p.H / p.Hkv;
  const int nk = key_count(p, b);
  const float c2 = p.scale * kLog2e;
  float dk[4][DP / 16] = {}, dv[4][DP / 16] = {};
  if (k0 < nk) {
    if (threadIdx.x < TM) okc[threadIdx.x] = key_ok(p, b, nk, k0 + threadIdx.x);
    __syncthreads();
    stage<T, DP, true, VEC, TM, NT>(sk, p.k, p, b, hk, k0, nk, okc);
    stage<T, DP, true, VEC, TM, NT>(sv, p.v, p, b, hk, k0, nk, okc);
    // the query heads that share this key head, one after another: a fixed order
    for (int g = 0; g < G; ++g)
      for (int r0 = 0; r0 < p.Lq; r0 += kT) {
        const int h = hk * G + g;
        __syncthreads();
        stage<T, DP, false, VEC, kT, NT>(sq, p.q, p, b, h, r0, p.Lq, nullptr);
        stage<T, DP, false, VEC, kT, NT>(sdo, p.dout, p, b, h, r0, p.Lq, nullptr);
        if (threadIdx.x < kT) {  // rows past the end weigh nothing
          const int row = r0 + threadIdx.x;
          const int64_t at = (b * p.H + h) * p.Lq + row;
          s_lse[threadIdx.x] = row < p.Lq ? p.lse2[at] : INFINITY;
          s_delta[threadIdx.x] = row < p.Lq ? p.delta[at] : 0.0f;
        }
        __syncthreads();
        float s[4][4] = {}, dp[4][4] = {};
        dot_tile<DP>(s, sk, sq, ty, tx);
        dot_tile<DP>(dp, sv, sdo, ty, tx);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float lse = s_lse[tx + 16 * j], delta = s_delta[tx + 16 * j];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float w = okc[4 * ty + i] ? exp2f(s[i][j] * c2 - lse) : 0.0f;
            const int at = (4 * ty + i) * (kT + 4) + tx + 16 * j;
            sp[at] = w;
            sds[at] = w * (dp[i][j] - delta);
          }
        }
        __syncwarp();
        gather_tile<DP>(dv, sp, sdo, ty, tx);
        gather_tile<DP>(dk, sds, sq, ty, tx);
      }
  }
  const float one[4] = {1.0f, 1.0f, 1.0f, 1.0f}, f[4] = {p.scale, p.scale, p.scale, p.scale};
  store_rows<T, DP>(p.dk, dk, f, p, b, p.Lk, p.Hkv, hk, k0, ty, tx);
  store_rows<T, DP>(p.dv, dv, one, p, b, p.Lk, p.Hkv, hk, k0, ty, tx);
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
  for (int d = lane; d < p.D; d += 32) a += io<T>::ld(o + d) * io<T>::ld(g + d);
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) a += __shfl_xor_sync(0xffffffffu, a, s);
  if (lane == 0) p.delta[(b * p.H + h) * p.Lq + t] = a;
}

template <typename T, int DP, bool VEC, int TM>
int launch_rows(const Params& p, int which, cudaStream_t st) {  // 0 forward, 1 dq, 2 dk and dv
  constexpr int NT = kTileThreads<TM>;
  const int64_t rows = which == 2 ? p.Lk : p.Lq, heads = which == 2 ? p.Hkv : p.H;
  const int64_t grid = (rows + TM - 1) / TM * heads * p.B;
  if (grid > 0x7fffffff) return HCLSM_ERR_SHAPE;
  if (grid == 0) return HCLSM_OK;
  const size_t bytes = which == 0   ? smem_bytes<DP, TM, 1, 2, 1>()
                       : which == 1 ? smem_bytes<DP, TM, 2, 2, 1>()
                                    : smem_bytes<DP, TM, 2, 2, 2>();
  auto f = which == 0 ? fwd_kernel<T, DP, VEC, TM> : which == 1 ? dq_kernel<T, DP, VEC, TM> : dkv_kernel<T, DP, VEC, TM>;
  if (!set_smem_limit(reinterpret_cast<const void*>(f), bytes)) return HCLSM_ERR_LAUNCH;
  return launch_pdl(f, (unsigned)grid, NT, bytes, st, p);
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
  auto view = [](const hclsm_view& v) { return View{v.p, v.sb, v.st, v.sh}; };
  p.q = view(a->q), p.k = view(a->k), p.v = view(a->v), p.dout = view(a->dout);
  p.o = a->o, p.dq = a->dq, p.dk = a->dk, p.dv = a->dv;
  p.lse2 = a->lse2;
  p.lens = a->lens, p.mask = a->mask, p.mask_sb = a->mask_sb;
  p.B = a->B, p.Lq = a->Lq, p.Lk = a->Lk, p.H = a->H, p.Hkv = a->Hkv, p.D = a->D;
  p.scale = a->scale;
  p.err = device_err_ptr();
  return p;
}

}  // namespace xattn
}  // namespace hclsm

using namespace hclsm;

// Few enough rows a key head that the 16-row products of the split form carry
// no padding to speak of, and operands it can read 16 bytes at a time.
static bool use_split(const xattn::Params& p, int dtype) {
  const int e = dtype == HCLSM_F32 ? 4 : 2;
  auto ok = [&](const xattn::View& v) {
    return reinterpret_cast<uintptr_t>(v.p) % 16 == 0 && v.sb * e % 16 == 0 && v.st * e % 16 == 0 && v.sh * e % 16 == 0;
  };
  return p.Lk > 0 && (int64_t)p.Lq * (p.H / p.Hkv) <= 16 && p.D % 32 == 0 && ok(p.k) && ok(p.v);
}

extern "C" size_t hclsm_xattn_fwd_workspace_size(const hclsm_xattn_args* a) {
  if (xattn::check(a)) return 0;
  const xattn::Params p = xattn::params(a);
  if (use_split(p, a->dtype)) return xattn::split_workspace(p, a->dtype);
  return a->dtype == HCLSM_BF16 && xattn::tc_ok(p, false) ? xattn::tc_workspace(p) : 0;
}

extern "C" int hclsm_xattn_fwd(const hclsm_xattn_args* a, void* ws, size_t ws_bytes, void* stream) {
  if (const int rc = xattn::check(a)) return rc;
  if ((int64_t)a->B * a->Lq == 0) return HCLSM_OK;
  if (!a->q.p || !a->o || (a->Lk > 0 && (!a->k.p || !a->v.p))) return HCLSM_ERR_NULL;
  const xattn::Params p = xattn::params(a);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (use_split(p, a->dtype)) {
    const size_t need = xattn::split_workspace(p, a->dtype);
    if (ws_bytes < need || (need && !ws)) return HCLSM_ERR_WORKSPACE;
    return xattn::split_fwd(p, a->dtype, ws, st);
  }
  if (a->dtype == HCLSM_BF16 && xattn::tc_ok(p, false)) {
    const size_t need = xattn::tc_workspace(p);
    if (ws_bytes < need || (need && !ws)) return HCLSM_ERR_WORKSPACE;
    return xattn::tc_fwd(p, ws, st);
  }
  return a->dtype == HCLSM_F32 ? xattn::dispatch<float>(p, false, st) : xattn::dispatch<__nv_bfloat16>(p, false, st);
}

static bool use_tc_bwd(const xattn::Params& p, int dtype) {
  auto al = [](const void* q) { return reinterpret_cast<uintptr_t>(q) % 16 == 0; };
  return dtype == HCLSM_BF16 && xattn::tc_ok(p, true) && al(p.dq) && al(p.dk) && al(p.dv);
}

extern "C" size_t hclsm_xattn_bwd_workspace_size(const hclsm_xattn_args* a) {
  if (xattn::check(a)) return 0;
  const xattn::Params p = xattn::params(a);
  return xattn::delta_bytes(p) + (a->dtype == HCLSM_BF16 ? xattn::tc_workspace(p) : 0);
}

extern "C" int hclsm_xattn_bwd(const hclsm_xattn_args* a, void* ws, size_t ws_bytes, void* stream) {
  if (const int rc = xattn::check(a)) return rc;
  if (a->B == 0) return HCLSM_OK;
  if (a->Lq > 0 && (!a->q.p || !a->o || !a->dout.p || !a->dq || !a->lse2)) return HCLSM_ERR_NULL;
  if (a->Lk > 0 && (!a->k.p || !a->v.p || !a->dk || !a->dv)) return HCLSM_ERR_NULL;
  if (ws_bytes < hclsm_xattn_bwd_workspace_size(a) || (a->Lq > 0 && !ws)) return HCLSM_ERR_WORKSPACE;
  xattn::Params p = xattn::params(a);
  p.delta = static_cast<float*>(ws);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (const int rc = xattn::launch_delta(p, a->dtype, st)) return rc;
  if (use_tc_bwd(p, a->dtype)) return xattn::tc_bwd(p, static_cast<char*>(ws) + xattn::delta_bytes(p), st);
  return a->dtype == HCLSM_F32 ? xattn::dispatch<float>(p, true, st) : xattn::dispatch<__nv_bfloat16>(p, true, st);
}
