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
// Both kernels move every byte once (writing re-reads a block from L1 after its
// maximum): the bound is HBM, at small sizes the launch.
#include "xattn.cuh"

namespace hclsm {
namespace kv8 {

constexpr int kThreads = 256;

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

template <typename T>
__device__ __forceinline__ void ld8(const T* p, float (&v)[8]) {
  if constexpr (sizeof(T) == 2) {
    const uint4 r = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  } else {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  }
}
template <typename T>
__device__ __forceinline__ void st8(T* p, const float (&v)[8]) {
  if constexpr (sizeof(T) == 2) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
  }
}

// One block of threads a touched cache block and head, blockIdx.y keys or values.
// The first one of a sequence also writes the tail, after it has read it.
template <typename T>
__global__ void __launch_bounds__(kThreads) write_kernel(const __grid_constant__ Params p) {
  __shared__ float red[kThreads / 32];
  __shared__ float s_max;
  pdl_wait();
  pdl_trigger();
  const int j = (int)(blockIdx.x % p.touched);
  const int64_t bh = blockIdx.x / p.touched;
  const int64_t b = bh / p.Hkv;
  const int hk = (int)(bh % p.Hkv), kv = blockIdx.y;
  const int start = p.start[b], count = p.count ? p.count[b] : p.n;
  // a request outside the cache or the new tokens writes nothing
  if (start < 0 || count < 0 || count > p.n || start > p.T - count) {
    if (threadIdx.x == 0) record_error(p.err, HCLSM_ERR_SHAPE);
    return;
  }
  if (count == 0) return;
  const int end = start + count, D = p.D, block = p.block, vecs = block * D / 8;
  const int blk = start / block + j, lastb = (end - 1) / block;
  if (blk > lastb) return;
  const xattn::View& xv = p.x[kv];
  const T* x = static_cast<const T*>(xv.p) + b * xv.sb + hk * xv.sh;
  T* tail = static_cast<T*>(p.tail[kv]) + bh * block * D;
  auto row = [&](int tok) { return tok >= start ? x + (int64_t)(tok - start) * xv.st : tail + (tok % block) * D; };
  if ((blk + 1) * block <= end) {
    float m = 0.0f;
    for (int i = threadIdx.x; i < vecs; i += kThreads) {
      float v[8];
      ld8(row(blk * block + i * 8 / D) + i * 8 % D, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float a = fabsf(v[e]);
        m = a <= 3.402823466e38f ? fmaxf(m, a) : INFINITY;  // INFINITY stays: fmaxf(inf, a) = inf
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < kThreads / 32; ++w) m = fmaxf(m, red[w]);
      const float s = m == INFINITY ? __int_as_float(0x7fc00000) : __fdiv_rn(m, 127.0f);
      s_max = s;
      p.scale[kv][bh * (p.T / block) + blk] = s;
    }
    __syncthreads();
    const float s = s_max;
    const bool fine = s > 0.0f;  // neither zero nor NaN
    int8_t* q = p.q[kv] + (bh * p.T + (int64_t)blk * block) * D;
    for (int i = threadIdx.x; i < vecs; i += kThreads) {
      float v[8];
      ld8(row(blk * block + i * 8 / D) + i * 8 % D, v);
      uint32_t w[2] = {0, 0};
      if (fine) {
#pragma unroll
        for (int e = 0; e < 8; ++e)  // |x / scale| can round past 127 where the scale is subnormal
          w[e >> 2] |= (uint32_t)(min(max(__float2int_rn(__fdiv_rn(v[e], s)), -127), 127) & 0xff) << (8 * (e & 3));
      }
      *reinterpret_cast<uint2*>(q + i * 8) = make_uint2(w[0], w[1]);
    }
  }
  if (j == 0 && end % block) {
    __syncthreads();  // the tail has been read
    const int t0 = max(start, lastb * block);
    for (int i = threadIdx.x; i < (end - t0) * D / 8; i += kThreads) {
      float v[8];
      const int tok = t0 + i * 8 / D, d = i * 8 % D;
      ld8(x + (int64_t)(tok - start) * xv.st + d, v);
      st8(tail + (tok % block) * D + d, v);
    }
  }
}

// 8 dims a thread, in the output's order.
template <typename T>
__global__ void __launch_bounds__(kThreads) read_kernel(const __grid_constant__ Params p) {
  pdl_wait();
  pdl_trigger();
  const int kv = blockIdx.y, vd = p.D / 8;
  const int64_t total = (int64_t)p.B * p.T * p.Hkv * vd;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += (int64_t)gridDim.x * kThreads) {
    const int d = (int)(i % vd) * 8;
    int64_t r = i / vd;
    const int hk = (int)(r % p.Hkv);
    r /= p.Hkv;
    const int t = (int)(r % p.T);
    const int64_t b = r / p.T, bh = b * p.Hkv + hk;
    const int n = p.count ? min(max(p.count[b], 0), p.T) : p.T;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.0f;
    if (t < n / p.block * p.block) {
      const float s = p.scale[kv][bh * (p.T / p.block) + t / p.block];
      const uint2 w = *reinterpret_cast<const uint2*>(p.q[kv] + (bh * p.T + t) * p.D + d);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = s * (float)(int8_t)((e < 4 ? w.x : w.y) >> (8 * (e & 3)));
    } else if (t < n) {
      ld8(static_cast<const T*>(p.tail[kv]) + (bh * p.block + t % p.block) * p.D + d, v);
    }
    st8(static_cast<T*>(p.out[kv]) + i * 8, v);
  }
}

size_t attn_workspace(const hclsm_kv8_cache* c, int Lq, int H);
int attn(const hclsm_kv8_cache* c, const hclsm_view* q, void* o, const int32_t* lens, int Lq, int H, float scale,
         void* ws, cudaStream_t st);

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

bool row16(const hclsm_view* v, int dtype) {
  const int e = dtype == HCLSM_F32 ? 4 : 2;
  return al16(v->p) && v->sb * e % 16 == 0 && v->st * e % 16 == 0 && v->sh * e % 16 == 0;
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
  if (!kv8::row16(k, c->dtype) || !kv8::row16(v, c->dtype)) return HCLSM_ERR_ALIGN;
  kv8::Params p = kv8::params(c);
  p.x[0] = xattn::View{k->p, k->sb, k->st, k->sh};
  p.x[1] = xattn::View{v->p, v->sb, v->st, v->sh};
  p.n = n, p.start = start, p.count = count;
  p.touched = (int)(((int64_t)n + c->block - 2) / c->block + 1);
  const int64_t grid = (int64_t)c->B * c->Hkv * p.touched;
  if (grid > 0x7fffffff) return HCLSM_ERR_SHAPE;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 g((unsigned)grid, 2);
  return c->dtype == HCLSM_F32 ? launch_pdl(kv8::write_kernel<float>, g, kv8::kThreads, 0, st, p)
                               : launch_pdl(kv8::write_kernel<__nv_bfloat16>, g, kv8::kThreads, 0, st, p);
}

extern "C" int hclsm_kv8_read(const hclsm_kv8_cache* c, void* k, void* v, const int32_t* lens, void* stream) {
  if (const int rc = kv8::check(c)) return rc;
  if ((int64_t)c->B * c->T == 0) return HCLSM_OK;
  if (!k || !v) return HCLSM_ERR_NULL;
  if (!kv8::al16(k) || !kv8::al16(v)) return HCLSM_ERR_ALIGN;
  kv8::Params p = kv8::params(c);
  p.out[0] = k, p.out[1] = v, p.count = lens;
  const int64_t blocks = ((int64_t)c->B * c->T * c->Hkv * (c->D / 8) + kv8::kThreads - 1) / kv8::kThreads;
  const int64_t most = (int64_t)num_sms() * 32;
  const dim3 g((unsigned)(blocks < most ? blocks : most), 2);
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
  return kv8::attn(c, q, o, lens, Lq, H, scale, ws, static_cast<cudaStream_t>(stream));
}
