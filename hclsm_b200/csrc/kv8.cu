// The 8-bit state cache: writing and reading back.
//
// A sequence's keys and values are held in blocks of `block` tokens a head.  A
// complete block is 8-bit integers and one fp32 scale,
//   scale = max |x| / 127,   q = round_half_even(x / scale),   x ~ q * scale,
// and the last, incomplete block stays in the inputs' own type (the tail), so
// every value is rounded to 8 bits exactly once, when its block fills, and never
// again when later tokens raise the block's maximum.  A block with a value that is
// not finite gets a NaN scale: what is read from it is NaN, not a wrong number.
//
// Both kernels move every byte once: the bound is HBM, at small sizes the launch.
// 8 x 2048 tokens, 6 heads of 64, bf16 (25 MB of states, 13 MB of integers): 16 to
// 18 us to write and 10 to 13 to read back from L2, one wave of blocks each.
#include "xattn.cuh"

namespace hclsm {
namespace kv8 {

constexpr int kThreads = 128;

struct Params {
  xattn::View x[2];  // new keys and values (B, n, Hkv, D)
  int8_t* q[2];
  float* scale[2];
  void* tail[2];
  const int32_t *start, *count;
  void* out[2];  // reading: (B, T, Hkv, D) dense
  int B, n, T, Hkv, D, block, touched;
  int* err;
};

// 8 elements as loaded, and as fp32.
template <typename T> struct Raw;
template <> struct Raw<__nv_bfloat16> {
  uint4 r;
  __device__ __forceinline__ void ld(const __nv_bfloat16* p) { r = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void st(__nv_bfloat16* p) const { *reinterpret_cast<uint4*>(p) = r; }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  __device__ __forceinline__ void set(const float (&v)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    r = make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <> struct Raw<float> {
  float4 a, b;
  __device__ __forceinline__ void ld(const float* p) {
    a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  }
  __device__ __forceinline__ void st(float* p) const {
    *reinterpret_cast<float4*>(p) = a, *reinterpret_cast<float4*>(p + 4) = b;
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  }
  __device__ __forceinline__ void set(const float (&v)[8]) {
    a = make_float4(v[0], v[1], v[2], v[3]), b = make_float4(v[4], v[5], v[6], v[7]);
  }
};

// The largest |x|; INFINITY for a value that is not finite, and it stays.
__device__ __forceinline__ float largest(float m, const float (&v)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float a = fabsf(v[e]);
    m = a <= 3.402823466e38f ? fmaxf(m, a) : INFINITY;
  }
  return m;
}
// 8 values over the scale, to the nearest integer (half to even); zeros where the scale is zero or NaN.  inv is the
// fp32 reciprocal of the scale: x * inv is within 3e-5 of the quotient, so only a value that lies nearer than 1e-4 to
// halfway between two integers needs the division itself (as do scales whose reciprocal is not exact enough).
__device__ __forceinline__ uint2 eight(const float (&v)[8], float s, float inv) {
  uint32_t w[2] = {0, 0};
  if (s > 0.0f) {
    float q[8];
    bool near = s < 1e-30f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      q[e] = v[e] * inv;
      near |= fabsf(q[e] - rintf(q[e])) > 0.4999f;
    }
    if (near) {
#pragma unroll
      for (int e = 0; e < 8; ++e) q[e] = __fdiv_rn(v[e], s);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)  // |x / scale| can round past 127 where the scale is subnormal
      w[e >> 2] |= (uint32_t)(min(max(__float2int_rn(q[e]), -127), 127) & 0xff) << (8 * (e & 3));
  }
  return make_uint2(w[0], w[1]);
}

// One warp a touched cache block of a head, keys or values: no barrier, and a block of
// up to 32 x 64 stays in registers between its maximum and its rounding.  The first
// one of a sequence also writes the tail, after it has read it.
constexpr int kHeld = 8;  // vectors of 8 a lane holds

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) write_kernel(const __grid_constant__ Params p) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, kv = blockIdx.y;
  const int64_t task = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  const int64_t bh = task / p.touched;
  const int j = (int)(task - bh * p.touched);
  const int64_t b = bh / p.Hkv;
  const int hk = (int)(bh - b * p.Hkv);
  if (b >= p.B) return;
  const int start = p.start[b], count = p.count ? p.count[b] : p.n;
  // a request outside the cache or the new tokens writes nothing
  if (start < 0 || count < 0 || count > p.n || start > p.T - count) {
    if (lane == 0) record_error(p.err, HCLSM_ERR_SHAPE);
    return;
  }
  if (count == 0) return;
  const int end = start + count, block = p.block, vecs = block * D / 8, mask = block - 1;  // block: a power of 2
  const int log = 31 - __clz(block), blk = (start >> log) + j, lastb = (end - 1) >> log;
  if (blk > lastb) return;
  const xattn::View& xv = p.x[kv];
  const T* x = static_cast<const T*>(xv.p) + b * xv.sb + hk * xv.sh;
  T* tail = static_cast<T*>(p.tail[kv]) + bh * block * D;
  auto at = [&](int i) {  // vector i of the cache block: among the new tokens, or in the tail
    const int tok = blk * block + i * 8 / D, d = i * 8 % D;
    return tok >= start ? x + (int64_t)(tok - start) * xv.st + d : tail + (tok & mask) * D + d;
  };
  if ((blk + 1) * block <= end) {
    float m = 0.0f, v[8];
    Raw<T> r[kHeld];
    const bool held = vecs <= 32 * kHeld;
    if (held) {
#pragma unroll
      for (int k = 0; k < kHeld; ++k)
        if (k * 32 + lane < vecs) r[k].ld(at(k * 32 + lane));
#pragma unroll
      for (int k = 0; k < kHeld; ++k)
        if (k * 32 + lane < vecs) {
          r[k].get(v);
          m = largest(m, v);
        }
    } else {
#pragma unroll 4
      for (int i = lane; i < vecs; i += 32) {
        Raw<T> t;
        t.ld(at(i));
        t.get(v);
        m = largest(m, v);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float s = m == INFINITY ? __int_as_float(0x7fc00000) : __fdiv_rn(m, 127.0f);
    const float inv = 1.0f / s;
    if (lane == 0) p.scale[kv][bh * (p.T >> log) + blk] = s;
    int8_t* q = p.q[kv] + (bh * p.T + (int64_t)blk * block) * D;
    if (held) {
#pragma unroll
      for (int k = 0; k < kHeld; ++k)
        if (k * 32 + lane < vecs) {
          r[k].get(v);
          *reinterpret_cast<uint2*>(q + (k * 32 + lane) * 8) = eight(v, s, inv);
        }
    } else {
#pragma unroll 4
      for (int i = lane; i < vecs; i += 32) {
        Raw<T> t;
        t.ld(at(i));
        t.get(v);
        *reinterpret_cast<uint2*>(q + i * 8) = eight(v, s, inv);
      }
    }
  }
  if (j == 0 && (end & mask)) {
    __syncwarp();  // the tail has been read
    const int t0 = max(start, lastb * block);
    if (lane == 0) p.scale[kv][bh * (p.T >> log) + lastb] = -1.0f;  // this block is in the tail
    for (int i = lane; i < (end - t0) * D / 8; i += 32) {
      const int tok = t0 + i * 8 / D, d = i * 8 % D;
      Raw<T> t;
      t.ld(x + (int64_t)(tok - start) * xv.st + d);
      t.st(tail + (tok & mask) * D + d);
    }
  }
}

// 8 dims a thread and item, in the output's order; blockIdx.y keys or values.
template <typename T>
__global__ void __launch_bounds__(kThreads) read_kernel(const __grid_constant__ Params p) {
  pdl_wait();
  pdl_trigger();
  const int kv = blockIdx.y;
  const uint32_t vd = p.D / 8, row = vd * p.Hkv;  // vectors of a token
  const int64_t b = blockIdx.z;
  const int n = p.count ? min(max(p.count[b], 0), p.T) : p.T;
  const int n8 = n / p.block * p.block;  // whole blocks below the length
  const uint32_t total = row * (uint32_t)p.T;  // of this sequence
  T* out = static_cast<T*>(p.out[kv]) + b * (int64_t)total * 8;
  for (uint32_t i = blockIdx.x * kThreads + threadIdx.x; i < total; i += gridDim.x * kThreads) {
    const uint32_t t = i / row, h = (i - t * row) / vd, d = (i - t * row - h * vd) * 8;
    const int64_t bh = b * p.Hkv + h;
    float v[8];
    Raw<T> r;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.0f;
    const float s = (int)t < n ? p.scale[kv][bh * (p.T / p.block) + t / (uint32_t)p.block] : 0.0f;
    if ((int)t < n8 || ((int)t < n && !(s < 0.0f))) {
      const uint2 w = *reinterpret_cast<const uint2*>(p.q[kv] + (bh * p.T + t) * p.D + d);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = s * (float)(int8_t)((e < 4 ? w.x : w.y) >> (8 * (e & 3)));
      r.set(v);
    } else if ((int)t < n) {
      r.ld(static_cast<const T*>(p.tail[kv]) + (bh * p.block + (t - n8)) * p.D + d);
    } else {
      r.set(v);
    }
    r.st(out + (int64_t)i * 8);
  }
}

size_t attn_workspace(const hclsm_kv8_cache* c, int Lq, int H);
int attn(const hclsm_kv8_cache* c, const hclsm_view* q, void* o, const int32_t* lens, int Lq, int H, float scale,
         void* ws, cudaStream_t st);

template <typename T>
int launch_write(const Params& p, dim3 g, cudaStream_t st) {
  switch (p.D) {
    case 32: return launch_pdl(write_kernel<T, 32>, g, kThreads, 0, st, p);
    case 64: return launch_pdl(write_kernel<T, 64>, g, kThreads, 0, st, p);
    case 96: return launch_pdl(write_kernel<T, 96>, g, kThreads, 0, st, p);
    default: return launch_pdl(write_kernel<T, 128>, g, kThreads, 0, st, p);
  }
}

bool al16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

int check(const hclsm_kv8_cache* c) {
  if (!c) return HCLSM_ERR_NULL;
  if (c->dtype != HCLSM_F32 && c->dtype != HCLSM_BF16) return HCLSM_ERR_DTYPE;
  if (c->B < 0 || c->Hkv < 1 || c->T < 0) return HCLSM_ERR_SHAPE;
  if (c->D != 32 && c->D != 64 && c->D != 96 && c->D != 128) return HCLSM_ERR_SHAPE;
  if (c->block != 16 && c->block != 32 && c->block != 64 && c->block != 128) return HCLSM_ERR_SHAPE;
  if (c->T % c->block) return HCLSM_ERR_SHAPE;
  if ((int64_t)c->B * c->T == 0) return HCLSM_OK;
  if (!c->k || !c->v || !c->k_scale || !c->v_scale || !c->k_tail || !c->v_tail) return HCLSM_ERR_NULL;
  if (!al16(c->k) || !al16(c->v) || !al16(c->k_tail) || !al16(c->v_tail)) return HCLSM_ERR_ALIGN;
  return HCLSM_OK;
}

bool row16(const xattn::View& v, int dtype) {
  const int e = dtype == HCLSM_F32 ? 4 : 2;
  return al16(v.p) && v.sb * e % 16 == 0 && v.st * e % 16 == 0 && v.sh * e % 16 == 0;
}

Params params(const hclsm_kv8_cache* c) {
  Params p = {};
  p.q[0] = c->k, p.q[1] = c->v;
  p.scale[0] = c->k_scale, p.scale[1] = c->v_scale;
  p.tail[0] = c->k_tail, p.tail[1] = c->v_tail;
  p.B = c->B, p.T = c->T, p.Hkv = c->Hkv, p.D = c->D, p.block = c->block;
  p.err = device_err_ptr();
  return p;
}

}  // namespace kv8
}  // namespace hclsm

using namespace hclsm;

extern "C" int hclsm_kv8_write(const hclsm_kv8_cache* c, const hclsm_view* k, const hclsm_view* v, int32_t n,
                               const int32_t* start, const int32_t* count, void* stream) {
  if (const int rc = kv8::check(c)) return rc;
  if (n < 0) return HCLSM_ERR_SHAPE;
  if ((int64_t)c->B * n == 0) return HCLSM_OK;
  if (!k || !v || !k->p || !v->p || !start) return HCLSM_ERR_NULL;
  if (c->T == 0) return HCLSM_ERR_SHAPE;
  kv8::Params p = kv8::params(c);
  p.x[0] = xattn::view(*k, c->B, n, c->Hkv), p.x[1] = xattn::view(*v, c->B, n, c->Hkv);
  if (!kv8::row16(p.x[0], c->dtype) || !kv8::row16(p.x[1], c->dtype)) return HCLSM_ERR_ALIGN;
  p.n = n, p.start = start, p.count = count;
  p.touched = (int)(((int64_t)n + c->block - 2) / c->block + 1);
  const int64_t grid = ((int64_t)c->B * c->Hkv * p.touched + kv8::kThreads / 32 - 1) / (kv8::kThreads / 32);
  if (grid > 0x7fffffff) return HCLSM_ERR_SHAPE;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 g((unsigned)grid, 2);
  return c->dtype == HCLSM_F32 ? kv8::launch_write<float>(p, g, st) : kv8::launch_write<__nv_bfloat16>(p, g, st);
}

extern "C" int hclsm_kv8_read(const hclsm_kv8_cache* c, void* k, void* v, const int32_t* lens, void* stream) {
  if (const int rc = kv8::check(c)) return rc;
  if ((int64_t)c->B * c->T == 0) return HCLSM_OK;
  if (!k || !v) return HCLSM_ERR_NULL;
  if (!kv8::al16(k) || !kv8::al16(v)) return HCLSM_ERR_ALIGN;
  kv8::Params p = kv8::params(c);
  p.out[0] = k, p.out[1] = v, p.count = lens;
  const int64_t total = (int64_t)c->T * c->Hkv * (c->D / 8);  // vectors of a sequence
  if (total > 0x7fffffff || c->B > 65535) return HCLSM_ERR_SHAPE;
  const int64_t blocks = (total + kv8::kThreads - 1) / kv8::kThreads, most = (int64_t)num_sms() * 16 / c->B + 1;
  const dim3 g((unsigned)(blocks < most ? blocks : most), 2, (unsigned)c->B);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return c->dtype == HCLSM_F32 ? launch_pdl(kv8::read_kernel<float>, g, kv8::kThreads, 0, st, p)
                               : launch_pdl(kv8::read_kernel<__nv_bfloat16>, g, kv8::kThreads, 0, st, p);
}

extern "C" size_t hclsm_kv8_attn_workspace_size(const hclsm_kv8_cache* c, int32_t Lq, int32_t H) {
  if (kv8::check(c) || Lq < 0 || H < 1 || H % c->Hkv) return 0;
  return kv8::attn_workspace(c, Lq, H);
}

extern "C" int hclsm_kv8_attn(const hclsm_kv8_cache* c, const hclsm_view* q, void* o, const int32_t* lens, int32_t Lq,
                              int32_t H, float scale, void* ws, size_t ws_bytes, void* stream) {
  if (const int rc = kv8::check(c)) return rc;
  if (Lq < 0 || H < 1 || H % c->Hkv || !(scale > 0.0f) || scale > 3.0e38f) return HCLSM_ERR_SHAPE;
  if ((int64_t)c->B * Lq == 0) return HCLSM_OK;
  if (c->T == 0) return HCLSM_ERR_SHAPE;
  if (!q || !q->p || !o) return HCLSM_ERR_NULL;
  const size_t need = kv8::attn_workspace(c, Lq, H);
  if (ws_bytes < need || (need && !ws)) return HCLSM_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(ws) % 16) return HCLSM_ERR_ALIGN;
  return kv8::attn(c, q, o, lens, Lq, H, scale, ws, static_cast<cudaStream_t>(stream));
}
