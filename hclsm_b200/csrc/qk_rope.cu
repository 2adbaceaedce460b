// Per-head norm of queries and keys with the position rotation in the same
// pass, forward and backward.
//
//   xh = x * r,  r = rsqrt(mean(x^2) + eps)   over the D dims of one head
//   z  = xh * w
//   y  = R(pos) z: the first `rot` dims as rot/2 pairs (a, b), each turned by
//        its angle: (a cos - b sin, b cos + a sin); the other dims pass
// and with u = R(pos)^T dy, g = u * w:
//   dw = sum over rows of u * xh
//   dx = r * (g - xh * mean(g * xh))
//
// Every element is read once and written once, about 10 (forward) and 25
// (backward) operations each, so the bound is HBM.  A lane holds 8 dims of a
// head (16 bytes of bf16, two 16-byte loads of fp32) and D / 8 lanes (rounded
// up to a power of two) a head, so a head's sums are a butterfly inside the
// warp and the half layout's partner dims are a shuffle away.  A warp takes
// the heads of ONE token, 32 / lanes-per-head at a time: the token's cos and
// sin (64 bytes a lane) are read once and stay in registers for all its heads.
// Queries and keys go in one launch, the first warps the queries'.
// 64 x 2048 tokens, 32 + 8 heads of 64, bf16: 284 to 293 us forward (4.6 to 4.7 TB/s; 69 %
// of the issue slots), 474 to 487 us backward (4.1 to 4.2 TB/s; 24 warps an SM keep too few
// loads in flight; 16 warps: 561 us).
#include "common.cuh"

namespace hclsm {
int* device_err_ptr();
int num_sms();

namespace rope {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kBwdPerSm = 3;  // resident blocks of the backward kernel

struct Side {
  const void* x;
  const void* dy;
  void* y;  // forward: y, backward: dx
  const float* w;
  const int32_t* pos;
  int64_t sb, st, sh;  // element strides of x (dy and y are dense)
  int L, H;
  int chunks;       // a token's heads are split over this many warps
  int64_t tasks;    // B * L * chunks
  int blocks;       // thread blocks that work on this side
  float* partial;   // (blocks, D) column sums of u * xh, or null
  float* dw;
};

struct Params {
  Side s[2];
  const float* cosv;
  const float* sinv;
  int P, rot, D, lph;  // lph: lanes per head
  float eps;
  int norm, inter;
  int* err;
};

// 8 elements as loaded, and as fp32.
template <typename T> struct Vec8;
template <> struct Vec8<__nv_bfloat16> {
  uint4 r;
  __device__ __forceinline__ void ld(const __nv_bfloat16* p) { r = __ldcs(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ void zero() { r = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void get(float2 (&v)[4]) const {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
  }
  // another lane's elements, or zeros
  __device__ __forceinline__ Vec8 from(int lane, bool some) const {
    Vec8 o;
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
    uint32_t q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      q[i] = __shfl_sync(0xffffffffu, w[i], lane);
      q[i] = some ? q[i] : 0u;
    }
    o.r = make_uint4(q[0], q[1], q[2], q[3]);
    return o;
  }
  static __device__ __forceinline__ void st(__nv_bfloat16* p, const float2 (&v)[4]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[i].x, v[i].y);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <> struct Vec8<float> {
  float4 a, b;
  __device__ __forceinline__ void ld(const float* p) {
    a = __ldcs(reinterpret_cast<const float4*>(p)), b = __ldcs(reinterpret_cast<const float4*>(p + 4));
  }
  __device__ __forceinline__ void zero() { a = b = make_float4(0, 0, 0, 0); }
  __device__ __forceinline__ void get(float2 (&v)[4]) const {
    v[0] = make_float2(a.x, a.y), v[1] = make_float2(a.z, a.w);
    v[2] = make_float2(b.x, b.y), v[3] = make_float2(b.z, b.w);
  }
  __device__ __forceinline__ Vec8 from(int lane, bool some) const {
    const float w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    float q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      q[i] = __shfl_sync(0xffffffffu, w[i], lane);
      q[i] = some ? q[i] : 0.0f;
    }
    Vec8 o;
    o.a = make_float4(q[0], q[1], q[2], q[3]), o.b = make_float4(q[4], q[5], q[6], q[7]);
    return o;
  }
  static __device__ __forceinline__ void st(float* p, const float2 (&v)[4]) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
    *reinterpret_cast<float4*>(p + 4) = make_float4(v[2].x, v[2].y, v[3].x, v[3].y);
  }
};
__device__ __forceinline__ void table8(const float* p, float (&v)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}

// The sum over a head's lanes.
template <int LPH>
__device__ __forceinline__ float head_sum(float v) {
#pragma unroll
  for (int o = LPH >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float2 swap(float2 v) { return make_float2(v.y, v.x); }

// One warp-task: the heads [h0, h1) of token t of batch b.
//
// With c and s the cosines and signed sines of the lane's dims, the rotation is
// y_i = c_i z_i + s_i z_p(i), p(i) the pair's other dim: in the same lane's pair
// (INTER) or, for the half layout, at the same place `hop` lanes away.  Forward:
// z = r w x, so w is folded into the angles once a token and r follows.  Backward:
// the transpose, with the sines' signs turned.
template <typename T, int LPH, bool INTER, bool BWD>
__device__ __forceinline__ void token(const Params& p, const Side& sd, uint32_t task, int lane, const float2 (&w)[4],
                                      float2 (&dw)[4]) {
  constexpr int U = sizeof(T) == 2 && !BWD ? 4 : 2;  // passes whose loads are in flight together
  constexpr int HPW = 32 / LPH;
  const uint32_t bt32 = task / (uint32_t)sd.chunks, b32 = bt32 / (uint32_t)sd.L;
  const int chunk = (int)(task - bt32 * (uint32_t)sd.chunks), t = (int)(bt32 - b32 * (uint32_t)sd.L);
  const int64_t bt = bt32, b = b32;
  const int hl = lane / LPH, d0 = (lane % LPH) * 8;
  const int per = (sd.H + sd.chunks - 1) / sd.chunks;
  const int h0 = chunk * per, h1 = min(sd.H, h0 + per);
  const bool dim_ok = d0 < p.D, in_rot = d0 < p.rot;
  const int half = p.rot >> 1, hop = half >> 3;
  const bool second = d0 >= half;
  const int partner = !INTER && in_rot ? (second ? lane - hop : lane + hop) : lane;
  const T* x = static_cast<const T*>(sd.x) + b * sd.sb + (int64_t)t * sd.st + (int64_t)hl * sd.sh + d0;
  const int64_t at = (bt * sd.H + hl) * p.D + d0;  // of the dense tensors
  const T* dy = static_cast<const T*>(sd.dy) + at;
  T* y = static_cast<T*>(sd.y) + at;
  Vec8<T> xr[U], gr[BWD ? U : 1];
  auto fetch = [&](int hb) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int h = hb + i * HPW;
      xr[i].zero();
      if (BWD) gr[BWD ? i : 0].zero();
      if (dim_ok && h + hl < h1) {
        xr[i].ld(x + h * sd.sh);
        if (BWD) gr[BWD ? i : 0].ld(dy + (int64_t)h * p.D);
      }
    }
  };
  fetch(h0);  // in flight while the position and then its angles arrive

  float2 c[4], s[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) c[i] = make_float2(1.0f, 1.0f), s[i] = make_float2(0.0f, 0.0f);
  if (p.rot > 0) {
    int pos = sd.pos ? sd.pos[bt] : t;
    const bool bad = pos < 0 || pos >= p.P;
    if (bad) {
      if (lane == 0) record_error(p.err, HCLSM_ERR_SHAPE);
      pos = 0;
    }
    if (in_rot) {
      const int64_t row = (int64_t)pos * half;
      const float sg = BWD ? -1.0f : 1.0f;
      if constexpr (INTER) {
        const float4 ca = *reinterpret_cast<const float4*>(p.cosv + row + (d0 >> 1));
        const float4 sa = *reinterpret_cast<const float4*>(p.sinv + row + (d0 >> 1));
        const float cv[4] = {ca.x, ca.y, ca.z, ca.w}, sv[4] = {sa.x, sa.y, sa.z, sa.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) c[i] = make_float2(cv[i], cv[i]), s[i] = make_float2(-sg * sv[i], sg * sv[i]);
      } else {
        float cv[8], sv[8];
        table8(p.cosv + row + d0 - (second ? half : 0), cv);
        table8(p.sinv + row + d0 - (second ? half : 0), sv);
        const float f = second ? sg : -sg;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          c[i] = make_float2(cv[2 * i], cv[2 * i + 1]), s[i] = make_float2(f * sv[2 * i], f * sv[2 * i + 1]);
      }
      if (bad) {  // a position outside the table: NaN, not another position's angle
#pragma unroll
        for (int i = 0; i < 4; ++i) c[i] = s[i] = make_float2(__int_as_float(0x7fc00000), __int_as_float(0x7fc00000));
      }
    }
  }
  if constexpr (!BWD) {
    if (sd.w) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float2 o = swap(w[i]);
        if (!INTER)
          o = make_float2(__shfl_sync(0xffffffffu, w[i].x, partner), __shfl_sync(0xffffffffu, w[i].y, partner));
        c[i] = mul2(c[i], w[i]), s[i] = mul2(s[i], o);
      }
    }
  }
  const float inv_d = 1.0f / (float)p.D;
  for (int hb = h0; hb < h1; hb += HPW * U) {  // warp-uniform trip count
    if (hb != h0) fetch(hb);
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (hb + i * HPW >= h1) break;  // warp-uniform
      const int h = hb + i * HPW;
      const bool ok = dim_ok && h + hl < h1;
      float2 v[4], o[4];
      xr[i].get(v);
      float r = 1.0f;
      if (p.norm) {
        float2 q = mul2(v[0], v[0]);
#pragma unroll
        for (int e = 1; e < 4; ++e) q = fma2(v[e], v[e], q);
        r = rsqrtf(head_sum<LPH>(q.x + q.y) * inv_d + p.eps);
      }
      const float2 rr = make_float2(r, r);
      if constexpr (!BWD) {
        if constexpr (INTER) {
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e] = in_rot ? swap(v[e]) : make_float2(0.0f, 0.0f);
        } else {
          xr[i].from(partner, in_rot).get(o);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = mul2(fma2(o[e], s[e], mul2(v[e], c[e])), rr);
        if (ok) Vec8<T>::st(y + (int64_t)h * p.D, v);
      } else {
        float2 u[4];
        gr[i].get(u);
        if constexpr (INTER) {
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e] = in_rot ? swap(u[e]) : make_float2(0.0f, 0.0f);
        } else {
          gr[i].from(partner, in_rot).get(o);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) u[e] = fma2(o[e], s[e], mul2(u[e], c[e]));
        if (p.norm) {
          float2 m = make_float2(0.0f, 0.0f);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            v[e] = mul2(v[e], rr);  // xh
            dw[e] = fma2(u[e], v[e], dw[e]);
            u[e] = mul2(u[e], w[e]);
            m = fma2(u[e], v[e], m);
          }
          const float mean = -head_sum<LPH>(m.x + m.y) * inv_d;
#pragma unroll
          for (int e = 0; e < 4; ++e) u[e] = mul2(fma2(v[e], make_float2(mean, mean), u[e]), rr);
        }
        if (ok) Vec8<T>::st(y + (int64_t)h * p.D, u);
      }
    }
  }
}

template <typename T, int LPH, bool INTER, bool BWD>
__global__ void __launch_bounds__(kThreads, BWD ? kBwdPerSm : 4) rope_kernel(const __grid_constant__ Params p) {
  __shared__ float red[BWD ? kWarps * 256 : 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool isk = blockIdx.x >= (unsigned)p.s[0].blocks;
  const Side& sd = p.s[isk ? 1 : 0];
  const int blk = (int)blockIdx.x - (isk ? p.s[0].blocks : 0);
  pdl_wait();
  pdl_trigger();
  const int d0 = (lane % LPH) * 8;
  float2 w[4], dw[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w[i] = make_float2(1.0f, 1.0f), dw[i] = make_float2(0.0f, 0.0f);
    if (sd.w && d0 < p.D) w[i] = make_float2(sd.w[d0 + 2 * i], sd.w[d0 + 2 * i + 1]);
  }
  for (int64_t task = (int64_t)blk * kWarps + warp; task < sd.tasks; task += (int64_t)sd.blocks * kWarps)
    token<T, LPH, INTER, BWD>(p, sd, (uint32_t)task, lane, w, dw);
  if constexpr (BWD) {
    if (sd.partial) {
      // the warp's heads, then the block's warps, both in a fixed order
#pragma unroll
      for (int o = LPH; o < 32; o <<= 1) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          dw[i].x += __shfl_xor_sync(0xffffffffu, dw[i].x, o);
          dw[i].y += __shfl_xor_sync(0xffffffffu, dw[i].y, o);
        }
      }
      if (lane < LPH && d0 < p.D) {
#pragma unroll
        for (int i = 0; i < 4; ++i) red[warp * 256 + d0 + 2 * i] = dw[i].x, red[warp * 256 + d0 + 2 * i + 1] = dw[i].y;
      }
      __syncthreads();
      for (int d = threadIdx.x; d < p.D; d += kThreads) {
        float a = 0.0f;
        for (int k = 0; k < kWarps; ++k) a += red[k * 256 + d];
        sd.partial[(int64_t)blk * p.D + d] = a;
      }
    }
  }
}

// The blocks' column sums, block blockIdx.x one side's; thread groups take every
// G-th row and are added in order.
__global__ void __launch_bounds__(1024) dw_kernel(const __grid_constant__ Params p) {
  __shared__ float red[1024];
  pdl_wait();
  const Side& sd = p.s[blockIdx.x];
  if (!sd.partial) return;
  const int D = p.D, G = 1024 / D;
  const int d = threadIdx.x % D, g = threadIdx.x / D;
  float a = 0.0f;
  if (g < G)
    for (int r = g; r < sd.blocks; r += G) a += sd.partial[(int64_t)r * D + d];
  red[threadIdx.x] = a;
  __syncthreads();
  if (g == 0) {
    for (int k = 1; k < G; ++k) a += red[k * D + d];
    sd.dw[d] = a;
  }
}

int lanes_per_head(int D) {
  int l = 4;
  while (l * 8 < D) l <<= 1;
  return l;
}

bool aligned(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// A token's heads go to one warp unless there are too few tokens to fill the
// GPU; then each warp takes as few as one pass over the lanes.
void plan(Side& s, int64_t B, int lph) {
  const int hpw = 32 / lph;
  int passes = (s.H + hpw - 1) / hpw;
  const int64_t tokens = B * s.L;
  int chunks = 1;
  while (chunks < passes && tokens * chunks < (int64_t)num_sms() * 64) chunks <<= 1;
  if (chunks > passes) chunks = passes;
  // whole passes to every chunk
  const int per = (passes + chunks - 1) / chunks * hpw;
  s.chunks = (s.H + per - 1) / per;
  s.tasks = tokens * s.chunks;
}

int check(const hclsm_rope_side* s, int64_t B, int P, int rot, bool bwd) {
  if (s->L < 0 || s->H < 1) return HCLSM_ERR_SHAPE;
  if (B * s->L == 0) return HCLSM_OK;
  if (!s->x || !s->y || (bwd && !s->dy)) return HCLSM_ERR_NULL;
  // an empty table has no row 0 either, which a position outside the table reads in its place
  if (rot > 0 && (P < 1 || (!s->pos && s->L > P))) return HCLSM_ERR_SHAPE;
  if (!aligned(s->x) || !aligned(s->y) || (bwd && !aligned(s->dy))) return HCLSM_ERR_ALIGN;
  return HCLSM_OK;
}

template <typename T, int LPH>
int launch(const Params& p, int grid, bool inter, bool bwd, cudaStream_t st) {
  if (bwd)
    return inter ? launch_pdl(rope_kernel<T, LPH, true, true>, grid, kThreads, 0, st, p)
                 : launch_pdl(rope_kernel<T, LPH, false, true>, grid, kThreads, 0, st, p);
  return inter ? launch_pdl(rope_kernel<T, LPH, true, false>, grid, kThreads, 0, st, p)
               : launch_pdl(rope_kernel<T, LPH, false, false>, grid, kThreads, 0, st, p);
}
template <typename T>
int launch(const Params& p, int grid, bool inter, bool bwd, cudaStream_t st) {
  switch (p.lph) {
    case 4: return launch<T, 4>(p, grid, inter, bwd, st);
    case 8: return launch<T, 8>(p, grid, inter, bwd, st);
    case 16: return launch<T, 16>(p, grid, inter, bwd, st);
    default: return launch<T, 32>(p, grid, inter, bwd, st);
  }
}

int run(const hclsm_rope_side* q, const hclsm_rope_side* k, const float* cosv, const float* sinv, int P, int rot,
        int64_t B, int D, float eps, int dtype, int flags, bool bwd, void* ws, size_t ws_bytes, void* stream) {
  if (dtype != HCLSM_F32 && dtype != HCLSM_BF16) return HCLSM_ERR_DTYPE;
  if (!q) return HCLSM_ERR_NULL;
  const bool inter = flags & HCLSM_ROPE_INTERLEAVED, norm = !(flags & HCLSM_ROPE_NO_NORM);
  if (B < 0 || D < 8 || D > 256 || D % 8 || rot < 0 || rot > D || rot % (inter ? 8 : 16) || P < 0)
    return HCLSM_ERR_SHAPE;
  if (rot > 0 && (!cosv || !sinv)) return HCLSM_ERR_NULL;
  if (rot > 0 && (!aligned(cosv) || !aligned(sinv))) return HCLSM_ERR_ALIGN;
  Params p = {};
  const hclsm_rope_side* in[2] = {q, k};
  const int e = dtype == HCLSM_F32 ? 4 : 2;
  p.lph = lanes_per_head(D);
  for (int i = 0; i < 2; ++i) {
    Side& s = p.s[i];
    s.chunks = 1;
    if (!in[i]) continue;
    if (const int rc = check(in[i], B, P, rot, bwd)) return rc;
    if (!norm && in[i]->w) return HCLSM_ERR_UNSUPPORTED;
    if ((in[i]->sb * e) % 16 || (in[i]->st * e) % 16 || (in[i]->sh * e) % 16) return HCLSM_ERR_ALIGN;
    s.x = in[i]->x, s.dy = in[i]->dy, s.y = in[i]->y, s.w = in[i]->w, s.pos = in[i]->pos;
    s.sb = in[i]->sb, s.st = in[i]->st, s.sh = in[i]->sh;
    s.L = in[i]->L, s.H = in[i]->H;
    if (B * s.L > 0) plan(s, B, p.lph);
    if (s.tasks > 0x7fffffff) return HCLSM_ERR_SHAPE;
    s.blocks = (int)((s.tasks + kWarps - 1) / kWarps);
  }
  if (bwd) {  // as many blocks as are resident, shared out by the heads of the two sides
    const int most = num_sms() * kBwdPerSm;
    const double work[2] = {(double)B * p.s[0].L * p.s[0].H, (double)B * p.s[1].L * p.s[1].H};
    int share = (int)(most * (work[1] / (work[0] + work[1] + 1e-9)) + 0.5);
    if (share < 1) share = 1;
    if (share > most - 1) share = most - 1;
    if (p.s[1].blocks > share) p.s[1].blocks = share;
    if (p.s[0].blocks > most - share) p.s[0].blocks = most - share;
  }
  for (int i = 0; i < 2; ++i) {
    Side& s = p.s[i];
    if (!in[i]) continue;
    if (bwd && in[i]->dw) {
      const size_t need = (size_t)s.blocks * D * sizeof(float);
      const size_t used = i ? (p.s[0].partial ? (size_t)p.s[0].blocks * D * sizeof(float) : 0) : 0;
      s.dw = in[i]->dw;
      if (need) {
        if (!ws || used + need > ws_bytes) return HCLSM_ERR_WORKSPACE;
        s.partial = reinterpret_cast<float*>(static_cast<char*>(ws) + used);
      }
    }
  }
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  for (int i = 0; i < 2; ++i)  // no rows: the weight's gradient is zero
    if (p.s[i].dw && p.s[i].blocks == 0 && cudaMemsetAsync(p.s[i].dw, 0, D * sizeof(float), st) != cudaSuccess)
      return HCLSM_ERR_LAUNCH;
  const int grid = p.s[0].blocks + p.s[1].blocks;
  if (grid == 0) return HCLSM_OK;
  p.cosv = cosv, p.sinv = sinv, p.P = P, p.rot = rot, p.D = D, p.eps = eps, p.norm = norm, p.inter = inter;
  p.err = device_err_ptr();
  const int rc = dtype == HCLSM_F32 ? launch<float>(p, grid, inter, bwd, st)
                                    : launch<__nv_bfloat16>(p, grid, inter, bwd, st);
  if (rc != HCLSM_OK || (!p.s[0].partial && !p.s[1].partial)) return rc;
  return launch_pdl(dw_kernel, 2, 1024, 0, st, p);
}

}  // namespace rope
}  // namespace hclsm

extern "C" int hclsm_qk_norm_rope(const hclsm_rope_side* q, const hclsm_rope_side* k, const float* cosv,
                                  const float* sinv, int32_t P, int32_t rot, int64_t B, int32_t D, float eps,
                                  int32_t dtype, int32_t flags, void* stream) {
  return hclsm::rope::run(q, k, cosv, sinv, P, rot, B, D, eps, dtype, flags, false, nullptr, 0, stream);
}

extern "C" size_t hclsm_qk_norm_rope_bwd_workspace_size(int32_t D) {
  if (D < 8 || D > 256) return 0;
  return ((size_t)hclsm::num_sms() * hclsm::rope::kBwdPerSm) * D * sizeof(float);
}

extern "C" int hclsm_qk_norm_rope_bwd(const hclsm_rope_side* q, const hclsm_rope_side* k, const float* cosv,
                                      const float* sinv, int32_t P, int32_t rot, int64_t B, int32_t D, float eps,
                                      int32_t dtype, int32_t flags, void* ws, size_t ws_bytes, void* stream) {
  return hclsm::rope::run(q, k, cosv, sinv, P, rot, B, D, eps, dtype, flags, true, ws, ws_bytes, stream);
}
