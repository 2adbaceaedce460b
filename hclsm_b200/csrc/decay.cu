// Linear attention with a decay for each head (decay.cuh has the mathematics): fp32 arithmetic on the FMA pipe (fp32
// tensors, and bf16 rows that a tensor map does not take), the join of segments, the single-token step and the C ABI.
#include <math.h>

#include "decay.cuh"

namespace hclsm {
namespace decay {

constexpr int kC = 64;        // tokens of a chunk
constexpr int kE = 64;        // value dims of a block
constexpr int kThreads = 256; // 16 x 16 threads, 4 x 4 values of a 64 x 64 product each
constexpr int kVs = kE + 4, kPs = kC + 4;  // row strides: 16-byte rows, 8 lanes on different banks

template <int DP> struct Smem {
  static constexpr int kXs = DP + 4;
  float x[kC * kXs], k[kC * kXs], v[kC * kVs], s[DP * kVs], p[kC * kPs];
  float w[kC];  // decays of the state's update
};

// rows [t0, t0 + 64) of a head into shared memory in fp32, zeros outside [0, n) and behind D
template <typename T, int W>
__device__ __forceinline__ void stage(float* dst, int stride, const View& v, int64_t base, int t0, int n, int d0, int D,
                                      int tid) {
  const T* p = static_cast<const T*>(v.p) + base;
  for (int i = tid; i < kC * (W / 4); i += kThreads) {
    const int r = i / (W / 4), d = i % (W / 4) * 4;
    float q[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (t0 + r < n) {
      const T* at = p + (int64_t)(t0 + r) * v.st + d0 + d;
      if (d0 + d + 4 <= D && reinterpret_cast<uintptr_t>(at) % (4 * sizeof(T)) == 0) {
        if constexpr (sizeof(T) == 4) {
          const float4 t = *reinterpret_cast<const float4*>(at);
          q[0] = t.x, q[1] = t.y, q[2] = t.z, q[3] = t.w;
        } else {
          const uint2 t = *reinterpret_cast<const uint2*>(at);
          q[0] = __uint_as_float(t.x << 16), q[1] = __uint_as_float(t.x & 0xffff0000u);
          q[2] = __uint_as_float(t.y << 16), q[3] = __uint_as_float(t.y & 0xffff0000u);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (d0 + d + e < D) q[e] = io<T>::ld(at + e);
      }
    }
    *reinterpret_cast<float4*>(dst + r * stride + d) = make_float4(q[0], q[1], q[2], q[3]);
  }
}

__device__ __forceinline__ float4 ld4(const float* p) { return *reinterpret_cast<const float4*>(p); }

// One block: 64 value dims of one segment of one head.  SUMS: the segment's own sum of k^T v alone.
// The state stays in registers (4 x 4 values a thread and 64 rows) between chunks; shared memory holds the copy that
// the queries read.  A chunk is 1.05 M multiplications of 8192 cycles at full rate, so the FMA pipe is the bound, and
// latency where blocks are few: 3 x 333 ragged tokens, 6 heads of 64, forward + backward 84 us (239 without segments).
template <typename T, int DP, bool SUMS>
__global__ void __launch_bounds__(kThreads) simt_kernel(const __grid_constant__ Batch bt) {
  const Pass& p = bt.p[blockIdx.x % bt.n];
  extern __shared__ __align__(16) unsigned char raw[];
  Smem<DP>& s = *reinterpret_cast<Smem<DP>*>(raw);
  constexpr int kXs = Smem<DP>::kXs, R = DP / 64;
  pdl_wait();
  pdl_trigger();
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const int tiles = (p.Dv + kE - 1) / kE;
  const uint32_t block = blockIdx.x / bt.n;
  const int e0 = (int)(block % tiles) * kE;
  const int seg = (int)(block / tiles % p.segs);
  const int64_t bh = block / tiles / p.segs;
  const int64_t b = bh / p.H;
  const int h = (int)(bh - b * p.H), r = p.rev ? 1 : 0;
  const int n = length(p, b);
  const float l2 = log2_decay(p.log_decay, h);
  const float2 whole = chunk_decay(p.log_decay, h, kC);
  const float factor = p.w;
  const int c_lo = seg * p.seg_chunks, c_end = min(c_lo + p.seg_chunks, chunks_of(p.L, kC));
  const int c_hi = min(c_end, chunks_of(n, kC));  // chunks with valid tokens
  const int64_t xb = b * p.x.sb + h * p.x.sh, kb = b * p.k.sb + h * p.k.sh, vb = b * p.v.sb + h * p.v.sh;
  T* y = static_cast<T*>(p.y) + (b * p.L * p.H + h) * (int64_t)p.Dv;

  float S[R][4][4];
  const int64_t sz = (int64_t)p.Dk * p.Dv;
#pragma unroll
  for (int q = 0; q < R; ++q)
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = q * 64 + ty * 4 + i, c = e0 + tx * 4 + e;
        float v = 0.0f;
        if (!SUMS && d < p.Dk && c < p.Dv) {
          if (p.segs > 1) v = p.part[(bh * p.segs + seg) * sz + (int64_t)d * p.Dv + c];
          else if (p.init) v = p.init[bh * sz + (p.init_t ? (int64_t)c * p.Dk + d : (int64_t)d * p.Dv + c)];
        }
        S[q][i][e] = v;
      }

  for (int it = 0; it < c_hi - c_lo; ++it) {
    const int c = p.rev ? c_hi - 1 - it : c_lo + it, t0 = c * kC;
    const int m = min(n - t0, kC);
    __syncthreads();
    stage<T, DP>(s.k, kXs, p.k, kb, t0, n, 0, p.Dk, tid);
    stage<T, kE>(s.v, kVs, p.v, vb, t0, n, e0, p.Dv, tid);
    if (!SUMS) {
      stage<T, DP>(s.x, kXs, p.x, xb, t0, n, 0, p.Dk, tid);
#pragma unroll
      for (int q = 0; q < R; ++q)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<float4*>(s.s + (q * 64 + ty * 4 + i) * kVs + tx * 4) =
              make_float4(S[q][i][0], S[q][i][1], S[q][i][2], S[q][i][3]);
    }
    if (tid < kC) {
      const int place = p.rev ? m - 1 - tid : tid;
      s.w[tid] = tid < m ? factor * exp2f(l2 * (float)(m - 1 - place + r)) : 0.0f;
    }
    __syncthreads();
    if (!SUMS) {
      {  // P = (X K^T) w g^|i - j|: rows 4 ty + i, columns tx + 16 j
        float a[4][4] = {};
#pragma unroll 4
        for (int d = 0; d < DP; d += 4) {
          float4 xr[4], kr[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) xr[i] = ld4(s.x + (ty * 4 + i) * kXs + d);
#pragma unroll
          for (int j = 0; j < 4; ++j) kr[j] = ld4(s.k + (tx + 16 * j) * kXs + d);
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              a[i][j] = fmaf(xr[i].x, kr[j].x, a[i][j]);
              a[i][j] = fmaf(xr[i].y, kr[j].y, a[i][j]);
              a[i][j] = fmaf(xr[i].z, kr[j].z, a[i][j]);
              a[i][j] = fmaf(xr[i].w, kr[j].w, a[i][j]);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int row = ty * 4 + i, col = tx + 16 * j, lag = p.rev ? col - row : row - col;
            s.p[row * kPs + col] = lag >= 0 ? a[i][j] * (factor * exp2f(l2 * (float)lag)) : 0.0f;
          }
      }
      __syncthreads();
      float o[4][4] = {};
#pragma unroll 4
      for (int d = 0; d < DP; d += 4) {  // x T
        float4 xr[4], sr[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) xr[i] = ld4(s.x + (ty * 4 + i) * kXs + d);
#pragma unroll
        for (int k = 0; k < 4; ++k) sr[k] = ld4(s.s + (d + k) * kVs + tx * 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float q[4] = {xr[i].x, xr[i].y, xr[i].z, xr[i].w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            o[i][0] = fmaf(q[k], sr[k].x, o[i][0]);
            o[i][1] = fmaf(q[k], sr[k].y, o[i][1]);
            o[i][2] = fmaf(q[k], sr[k].z, o[i][2]);
            o[i][3] = fmaf(q[k], sr[k].w, o[i][3]);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = ty * 4 + i, place = p.rev ? m - 1 - row : row;
        const float lead = row < m ? exp2f(l2 * (float)(place + 1 - r)) : 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][e] *= lead;
      }
#pragma unroll 4
      for (int j = 0; j < kC; j += 4) {  // P v
        float4 pr[4], vr[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) pr[i] = ld4(s.p + (ty * 4 + i) * kPs + j);
#pragma unroll
        for (int k = 0; k < 4; ++k) vr[k] = ld4(s.v + (j + k) * kVs + tx * 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float q[4] = {pr[i].x, pr[i].y, pr[i].z, pr[i].w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            o[i][0] = fmaf(q[k], vr[k].x, o[i][0]);
            o[i][1] = fmaf(q[k], vr[k].y, o[i][1]);
            o[i][2] = fmaf(q[k], vr[k].z, o[i][2]);
            o[i][3] = fmaf(q[k], vr[k].w, o[i][3]);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = ty * 4 + i;
        if (row >= m) continue;
        T* out = y + (int64_t)(t0 + row) * p.H * p.Dv + e0 + tx * 4;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (e0 + tx * 4 + e < p.Dv) io<T>::st(out + e, p.f * o[i][e]);
      }
    }
    const bool more = SUMS || it + 1 < c_hi - c_lo || (p.segs == 1 && p.last);
    if (more) {
      const float2 g = m == kC ? whole : chunk_decay(p.log_decay, h, m);
#pragma unroll
      for (int q = 0; q < R; ++q) {
        float a[4][4] = {};
#pragma unroll 8
        for (int j = 0; j < kC; ++j) {
          const float4 kr = ld4(s.k + j * kXs + q * 64 + ty * 4), vr = ld4(s.v + j * kVs + tx * 4);
          const float w = s.w[j];
          const float kk[4] = {kr.x * w, kr.y * w, kr.z * w, kr.w * w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            a[i][0] = fmaf(kk[i], vr.x, a[i][0]);
            a[i][1] = fmaf(kk[i], vr.y, a[i][1]);
            a[i][2] = fmaf(kk[i], vr.z, a[i][2]);
            a[i][3] = fmaf(kk[i], vr.w, a[i][3]);
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) S[q][i][e] = fmaf(S[q][i][e], g.x, fmaf(S[q][i][e], g.y, a[i][e]));
      }
    }
  }
  if (SUMS || (p.segs == 1 && p.last)) {
    float* out = SUMS ? p.part + (bh * p.segs + seg) * sz : p.last + bh * sz;
#pragma unroll
    for (int q = 0; q < R; ++q)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int d = q * 64 + ty * 4 + i, c = e0 + tx * 4 + e;
          if (d < p.Dk && c < p.Dv) out[(int64_t)d * p.Dv + c] = S[q][i][e];
        }
  }
  if (!SUMS)  // rows behind the length
    for (int64_t t = max(c_lo * kC, n) + (int64_t)ty, end = min((int64_t)c_end * kC, (int64_t)p.L); t < end; t += 16)
      for (int e = tx; e < min(kE, p.Dv - e0); e += 16) io<T>::st(y + t * p.H * p.Dv + e0 + e, 0.0f);
}

// The segments' sums become their first states; the state behind the last one (in the pass's order) goes to `last`.
// Eight sums are asked for at a time, so a thread waits for memory once in eight segments.
__global__ void __launch_bounds__(128) join_kernel(const __grid_constant__ Batch bt, int chunk) {
  const Pass& p = bt.p[blockIdx.x % bt.n];
  __shared__ float2 s_g[2];
  pdl_wait();
  pdl_trigger();
  const int64_t sz = (int64_t)p.Dk * p.Dv;
  const int64_t per = (sz + 127) / 128;
  const int64_t block = blockIdx.x / bt.n, bh = block / per, i = block % per * 128 + threadIdx.x;
  const int64_t b = bh / p.H;
  const int h = (int)(bh - b * p.H), n = length(p, b), span = p.seg_chunks * chunk;
  const bool in = i < sz;
  const int segs = p.segs, step = p.rev ? -1 : 1, first = p.rev ? segs - 1 : 0;
  float* at = p.part + (bh * segs + first) * sz + i;
  const int64_t by = step * sz;
  float sum[8];
  auto ask = [&](int it) {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (in && it + k < segs) sum[k] = at[(it + k) * by];
  };
  ask(0);  // on their way while the decays, of a whole segment and of the incomplete one, are formed
  if (threadIdx.x < 2) s_g[threadIdx.x] = chunk_decay(p.log_decay, h, threadIdx.x ? n % span : span);
  __syncthreads();
  if (!in) return;
  float v = 0.0f;
  if (p.init) v = p.init[bh * sz + (p.init_t ? i % p.Dv * p.Dk + i / p.Dv : i)];
  const float2 whole = s_g[0], cut_off = s_g[1];
  for (int it = 0; it < segs; it += 8) {
    if (it > 0) ask(it);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int64_t m = n - (int64_t)(first + step * (it + k)) * span;  // tokens from this segment on
      if (it + k < segs) at[(it + k) * by] = v;
      if (it + k < segs && m > 0) {  // not behind the length
        const float2 g = m >= span ? whole : cut_off;
        v = fmaf(v, g.x, fmaf(v, g.y, sum[k]));
      }
    }
  }
  if (p.last) p.last[bh * sz + i] = v;
}

int join(const Batch& b, int chunk, cudaStream_t st) {
  const Pass& p = b.p[0];
  const int64_t grid = (int64_t)b.n * p.B * p.H * (((int64_t)p.Dk * p.Dv + 127) / 128);
  if (grid > 0x7fffffff) return HCLSM_ERR_SHAPE;
  return launch_pdl(join_kernel, (unsigned)grid, 128, 0, st, b, chunk);
}

template <typename T, int DP, bool SUMS>
int launch_simt(const Batch& b, cudaStream_t st) {
  auto fn = simt_kernel<T, DP, SUMS>;
  if (!set_smem_limit(reinterpret_cast<const void*>(fn), sizeof(Smem<DP>))) return HCLSM_ERR_LAUNCH;
  const Pass& p = b.p[0];
  const int64_t grid = (int64_t)b.n * p.B * p.H * p.segs * ((p.Dv + kE - 1) / kE);
  if (grid > 0x7fffffff) return HCLSM_ERR_SHAPE;
  return launch_pdl(fn, (unsigned)grid, kThreads, sizeof(Smem<DP>), st, b);
}

template <typename T>
int simt_run(const Batch& b, cudaStream_t st) {
  const Pass& p = b.p[0];
  if (p.segs > 1) {
    if (const int rc = p.Dk <= 64 ? launch_simt<T, 64, true>(b, st) : launch_simt<T, 128, true>(b, st)) return rc;
    if (const int rc = join(b, kC, st)) return rc;
  }
  return p.Dk <= 64 ? launch_simt<T, 64, false>(b, st) : launch_simt<T, 128, false>(b, st);
}

void simt_cut(Batch& b) {
  const Pass& p = b.p[0];
  cut(b, kC, 1.6f, 1.1f, 1.0f, 0.0f,
      (int64_t)b.n * p.B * p.H * ((p.Dv + kE - 1) / kE), (int64_t)num_sms() * (p.Dk <= 64 ? 2 : 1));
}

// ---- one token -------------------------------------------------------------------------------
// A block a head: V = 4 (or 1) value dims and every kThreads / (Dv / V)-th row of the state a thread.
// The decay is in two fp32 parts, as the chunks' are: one fp32 number is up to 2^-25 off it, at every token the same way, so that
// e^-1e-6 a token would forget 1.3 % too slowly.  Each value of the state is read and written once; the bound is memory: 256 x 16 states of 128 x 128 in 84 us, 6.4 TB/s.
struct Step {
  const void *q, *k, *v;
  void* o;
  const float *log_decay, *s0;
  float* s1;
  const uint8_t* active;
  int64_t qb, qh, kb, kh, vb, vh;  // strides in elements
  int B, H, Dk, Dv;
  float scale;
};

constexpr int kStepThreads = 256;

template <typename T, int V>
__global__ void __launch_bounds__(kStepThreads) step_kernel(const __grid_constant__ Step p) {
  __shared__ float sq[128], sk[128], sv[128], red[kStepThreads * V];
  __shared__ float2 s_g;
  pdl_wait();
  pdl_trigger();
  const int64_t bh = blockIdx.x, b = bh / p.H;
  const int h = (int)(bh - b * p.H), tid = threadIdx.x;
  const bool on = !p.active || p.active[b];
  const int cols = (p.Dv + V - 1) / V, groups = kStepThreads / cols;
  const int e = tid % cols * V, g0 = tid / cols;
  const float* s0 = p.s0 + bh * p.Dk * p.Dv;
  float* s1 = p.s1 + bh * p.Dk * p.Dv;
  T* o = static_cast<T*>(p.o) + bh * p.Dv;
  if (!on) {
    if (s0 != s1)
      for (int i = tid; i < p.Dk * p.Dv; i += kStepThreads) s1[i] = s0[i];
    for (int i = tid; i < p.Dv; i += kStepThreads) io<T>::st(o + i, 0.0f);
    return;
  }
  if (tid < p.Dk) {
    sq[tid] = io<T>::ld(static_cast<const T*>(p.q) + b * p.qb + h * p.qh + tid);
    sk[tid] = io<T>::ld(static_cast<const T*>(p.k) + b * p.kb + h * p.kh + tid);
  }
  if (tid < p.Dv) sv[tid] = io<T>::ld(static_cast<const T*>(p.v) + b * p.vb + h * p.vh + tid);
  if (tid == kStepThreads - 1) s_g = chunk_decay(p.log_decay, h, 1);
  __syncthreads();
  const float2 g = s_g;
  float acc[V] = {};
  if (g0 < groups) {
    // eight rows asked for before the first is written: s1 may be s0, which keeps a load behind a store
    for (int d0 = g0; d0 < p.Dk; d0 += 8 * groups) {
      float s[8][V];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int d = d0 + i * groups;
        if (d >= p.Dk) continue;
        if constexpr (V == 4) {
          const float4 t = __ldcs(reinterpret_cast<const float4*>(s0 + d * p.Dv + e));
          s[i][0] = t.x, s[i][1] = t.y, s[i][2] = t.z, s[i][3] = t.w;
        } else {
          s[i][0] = s0[d * p.Dv + e];
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int d = d0 + i * groups;
        if (d >= p.Dk) continue;
#pragma unroll
        for (int k = 0; k < V; ++k) {
          s[i][k] = fmaf(s[i][k], g.x, fmaf(s[i][k], g.y, sk[d] * sv[e + k]));
          acc[k] = fmaf(sq[d], s[i][k], acc[k]);
        }
        if constexpr (V == 4)
          __stcs(reinterpret_cast<float4*>(s1 + d * p.Dv + e), make_float4(s[i][0], s[i][1], s[i][2], s[i][3]));
        else
          s1[d * p.Dv + e] = s[i][0];
      }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) red[(g0 * cols + e / V) * V + i] = acc[i];
  }
  __syncthreads();
  if (tid < p.Dv) {
    float sum = 0.0f;
    for (int q = 0; q < groups; ++q) sum += red[q * cols * V + tid];
    io<T>::st(o + tid, p.scale * sum);
  }
}

// ---- host ----------------------------------------------------------------------------------
int check(const hclsm_decay_args* a) {
  if (!a) return HCLSM_ERR_NULL;
  if (a->dtype != HCLSM_F32 && a->dtype != HCLSM_BF16) return HCLSM_ERR_DTYPE;
  if (a->B < 0 || a->L < 0 || a->H < 1 || a->D < 1 || a->D > 128 || a->Dv < 1 || a->Dv > 128) return HCLSM_ERR_SHAPE;
  if (!(a->scale > 0.0f) || a->scale > 3.0e38f) return HCLSM_ERR_SHAPE;
  return HCLSM_OK;
}

Pass base(const hclsm_decay_args* a) {
  Pass p = {};
  p.log_decay = a->log_decay, p.lens = a->lens;
  p.B = a->B, p.L = a->L, p.H = a->H;
  p.w = 1.0f, p.f = a->scale;
  p.err = device_err_ptr();
  return p;
}
View view(const hclsm_decay_args* a, const hclsm_view& v) { return xattn::view(v, a->B, a->L, a->H); }

Pass forward(const hclsm_decay_args* a) {
  Pass p = base(a);
  p.x = view(a, a->q), p.k = view(a, a->k), p.v = view(a, a->v), p.y = a->o;
  p.Dk = a->D, p.Dv = a->Dv, p.init = a->s0, p.last = a->s1;
  return p;
}
Pass grad_q(const hclsm_decay_args* a) {
  Pass p = base(a);
  p.x = view(a, a->dout), p.k = view(a, a->v), p.v = view(a, a->k), p.y = a->dq;
  p.Dk = a->Dv, p.Dv = a->D, p.init = a->s0, p.init_t = 1;
  return p;
}
Pass grad_v(const hclsm_decay_args* a) {
  Pass p = base(a);
  p.x = view(a, a->k), p.k = view(a, a->q), p.v = view(a, a->dout), p.y = a->dv;
  p.Dk = a->D, p.Dv = a->Dv, p.rev = 1;
  p.init = a->ds1, p.last = a->ds0, p.w = a->scale, p.f = 1.0f;
  return p;
}
Pass grad_k(const hclsm_decay_args* a) {
  Pass p = base(a);
  p.x = view(a, a->v), p.k = view(a, a->dout), p.v = view(a, a->q), p.y = a->dk;
  p.Dk = a->Dv, p.Dv = a->D, p.rev = 1;
  p.init = a->ds1, p.init_t = 1, p.w = a->scale, p.f = 1.0f;
  return p;
}

// The passes of a call, those of the same sizes together.
Batch forward_batch(const hclsm_decay_args* a) {
  Batch b = {};
  b.p[b.n++] = forward(a);
  return b;
}
int backward_batches(const hclsm_decay_args* a, Batch (&b)[2]) {
  b[0] = b[1] = Batch{};
  b[0].p[b[0].n++] = grad_k(a);
  b[0].p[b[0].n++] = grad_q(a);
  Batch& v = a->D == a->Dv ? b[0] : b[1];
  v.p[v.n++] = grad_v(a);
  return b[1].n ? 2 : 1;
}
// Cut into segments; the workspace's bytes, with the parts placed in it.
size_t plan(Batch& b, int dtype, void* ws) {
  if (dtype == HCLSM_BF16 && tc_ok(b)) tc_cut(b);
  else simt_cut(b);
  return parts(b, ws);
}
int run(const Batch& b, int dtype, cudaStream_t st) {
  if (dtype == HCLSM_BF16 && tc_ok(b)) return tc_run(b, st);
  return dtype == HCLSM_F32 ? simt_run<float>(b, st) : simt_run<__nv_bfloat16>(b, st);
}

// Without tokens the state passes through.
int only_state(float* to, const float* from, size_t n, cudaStream_t st) {
  if (!to || n == 0) return HCLSM_OK;
  const cudaError_t e = from ? cudaMemcpyAsync(to, from, n * sizeof(float), cudaMemcpyDeviceToDevice, st)
                             : cudaMemsetAsync(to, 0, n * sizeof(float), st);
  return e == cudaSuccess ? HCLSM_OK : HCLSM_ERR_LAUNCH;
}

}  // namespace decay
}  // namespace hclsm

using namespace hclsm;

extern "C" size_t hclsm_decay_attn_fwd_workspace_size(const hclsm_decay_args* a) {
  if (decay::check(a)) return 0;
  decay::Batch b = decay::forward_batch(a);
  return decay::plan(b, a->dtype, nullptr);
}

extern "C" int hclsm_decay_attn_fwd(const hclsm_decay_args* a, void* ws, size_t ws_bytes, void* stream) {
  if (const int rc = decay::check(a)) return rc;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a->B == 0) return HCLSM_OK;
  if (a->L == 0) return decay::only_state(a->s1, a->s0, (size_t)a->B * a->H * a->D * a->Dv, st);
  if (!a->q.p || !a->k.p || !a->v.p || !a->o || !a->log_decay) return HCLSM_ERR_NULL;
  decay::Batch b = decay::forward_batch(a);
  const size_t need = decay::plan(b, a->dtype, ws);
  if (ws_bytes < need || (need && !ws)) return HCLSM_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(ws) % 16) return HCLSM_ERR_ALIGN;
  return decay::run(b, a->dtype, st);
}

extern "C" size_t hclsm_decay_attn_bwd_workspace_size(const hclsm_decay_args* a) {
  if (decay::check(a)) return 0;
  decay::Batch b[2];
  const int n = decay::backward_batches(a, b);
  size_t most = 0;
  for (int i = 0; i < n; ++i) {
    const size_t need = decay::plan(b[i], a->dtype, nullptr);
    most = need > most ? need : most;
  }
  return most;
}

extern "C" int hclsm_decay_attn_bwd(const hclsm_decay_args* a, void* ws, size_t ws_bytes, void* stream) {
  if (const int rc = decay::check(a)) return rc;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a->B == 0) return HCLSM_OK;
  if (a->L == 0) return decay::only_state(a->ds0, a->ds1, (size_t)a->B * a->H * a->D * a->Dv, st);
  if (!a->q.p || !a->k.p || !a->v.p || !a->dout.p || !a->dq || !a->dk || !a->dv || !a->log_decay)
    return HCLSM_ERR_NULL;
  const size_t need = hclsm_decay_attn_bwd_workspace_size(a);
  if (ws_bytes < need || (need && !ws)) return HCLSM_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(ws) % 16) return HCLSM_ERR_ALIGN;
  decay::Batch b[2];
  const int n = decay::backward_batches(a, b);
  for (int i = 0; i < n; ++i) {
    decay::plan(b[i], a->dtype, ws);
    if (const int rc = decay::run(b[i], a->dtype, st)) return rc;
  }
  return HCLSM_OK;
}

extern "C" int hclsm_decay_attn_step(const hclsm_decay_args* a, const uint8_t* active, void* stream) {
  if (const int rc = decay::check(a)) return rc;
  if (a->B == 0) return HCLSM_OK;
  if (!a->q.p || !a->k.p || !a->v.p || !a->o || !a->log_decay || !a->s0 || !a->s1) return HCLSM_ERR_NULL;
  decay::Step p = {};
  p.q = a->q.p, p.k = a->k.p, p.v = a->v.p, p.o = a->o;
  p.qb = a->q.sb, p.qh = a->q.sh, p.kb = a->k.sb, p.kh = a->k.sh, p.vb = a->v.sb, p.vh = a->v.sh;
  p.log_decay = a->log_decay, p.s0 = a->s0, p.s1 = a->s1, p.active = active;
  p.B = a->B, p.H = a->H, p.Dk = a->D, p.Dv = a->Dv, p.scale = a->scale;
  const int64_t grid = (int64_t)a->B * a->H;
  if (grid > 0x7fffffff) return HCLSM_ERR_SHAPE;
  const bool four = a->Dv % 4 == 0 && reinterpret_cast<uintptr_t>(a->s0) % 16 == 0 &&
                    reinterpret_cast<uintptr_t>(a->s1) % 16 == 0;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 g((unsigned)grid), t(decay::kStepThreads);
  if (a->dtype == HCLSM_F32)
    return four ? launch_pdl(decay::step_kernel<float, 4>, g, t, 0, st, p)
                : launch_pdl(decay::step_kernel<float, 1>, g, t, 0, st, p);
  return four ? launch_pdl(decay::step_kernel<__nv_bfloat16, 4>, g, t, 0, st, p)
              : launch_pdl(decay::step_kernel<__nv_bfloat16, 1>, g, t, 0, st, p);
}
