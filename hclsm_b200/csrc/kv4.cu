// The paged 4-bit state cache: writing, reading and the C ABI (kv4.cuh has the format, kv4_attn.cu the attention).
// Both kernels move each byte once; eight values a thread, four threads a group.  8 x 2048 tokens, 6 heads of 64, 0.75 of
// them there, written and read back: 25 us with their slots; a wave of blocks each, bound by their start and by issue.
#include "kv4.cuh"

namespace hclsm {
namespace kv4 {

constexpr int kThreads = 256;

template <typename T> __device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
    const uint4 r = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
template <typename T> __device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// The nearest whole number of x / s in [-8, 7] (halves to even), plus 8.  inv is the fp32 reciprocal of s, so x * inv
// may lie on the wrong side of the middle between two codes (its floor k is off only next to a whole number, where
// k + 1/2 separates as well); the sign of x - (k + 1/2) s does not lie: fma rounds once.
__device__ __forceinline__ uint32_t code(float x, float s, float inv) {
  const float k = fminf(fmaxf(floorf(x * inv), -9.0f), 8.0f);
  const float over = fmaf(-(k + 0.5f), s, x);
  const int i = (int)k;
  const bool above = s < 0.0f ? over < 0.0f : over > 0.0f;
  return (uint32_t)(min(max(i + ((above || (over == 0.0f && (i & 1))) ? 1 : 0), -8), 7) + 8);
}
// The codes of eight values, four dims a word: adding 1.5 * 2^23 to the quotient rounds it to a whole number (halves to
// even), which the low bits then are.
// bf16 values: x * inv and one correction is the quotient itself where fp32 holds it, halves of whole numbers among
// them, and a quotient of two 8-bit numbers is no nearer to such a half than 2^-17 of it without being it.
// fp32 values may be: there x * inv, within 2e-6 of the quotient, decides but for a value within 1e-4 of a half, which
// goes through code(), as does a group whose scale is too small for a reciprocal.
template <bool EXACT> __device__ __forceinline__ void codes(const float (&v)[8], float s, uint32_t (&run)[2]) {
  const float inv = 1.0f / s;
  int r[8];
  float far = fabsf(s) < 1e-30f ? 1.0f : 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float q = v[e] * inv;
    if (EXACT) q = fmaf(fmaf(-q, s, v[e]), inv, q);
    const float t = q + 12582912.0f;
    if (!EXACT) far = fmaxf(far, fabsf(q + (12582912.0f - t)));
    r[e] = min(__float_as_int(t), 0x4b400000 + 7);
  }
  if (far < 0.4999f) {
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      uint32_t x = (uint32_t)r[4 * w + 3];
#pragma unroll
      for (int e = 2; e >= 0; --e) x = x * 16u + (uint32_t)r[4 * w + e];
      run[w] = x - 0x4b400000u * 0x1111u + 0x8888u;
    }
    return;
  }
  const float f = fabsf(s) < 1e-30f ? 0x1p64f : 1.0f, sf = s * f, inv_f = 1.0f / sf;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    run[w] = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) run[w] |= code(v[4 * w + e] * f, sf, inv_f) << (4 * e);
  }
}

struct Write {
  Cache c;
  xattn::View x[2];
  const int32_t* slots;
  int n;
  uint32_t total;  // threads with work
  int* err;
};

// blockIdx.y: keys or values.  Eight lanes hold 64 dims of a token (four the 32 behind them): the largest value of each
// group by shuffles, and each pair of lanes with the same dims of the two groups makes whole words.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) write_kernel(const __grid_constant__ Write p) {
  pdl_wait();
  pdl_trigger();
  constexpr int lanes = D / 8;
  const int kv = blockIdx.y;
  const uint32_t i = blockIdx.x * kThreads + threadIdx.x;
  const bool in = i < p.total;
  const uint32_t row = in ? i / lanes : 0, part = in ? i % lanes : 0;
  const uint32_t token = row / (uint32_t)p.c.Hkv, h = row - token * (uint32_t)p.c.Hkv;
  const uint32_t b = token / (uint32_t)p.n, t = token - b * (uint32_t)p.n;
  const int slot = in ? p.slots[token] : -1;
  const bool fits = slot >= 0 && (slot >> p.c.log_page) < p.c.pages;
  if (slot >= 0 && !fits) record_error(p.err, HCLSM_ERR_SHAPE);
  float v[8] = {};
  if (fits)
    load8(static_cast<const T*>(p.x[kv].p) + (int64_t)b * p.x[kv].sb + (int64_t)t * p.x[kv].st + (int64_t)h * p.x[kv].sh + part * 8,
          v);
  float hi = v[0], lo = v[0], finite = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    hi = fmaxf(hi, v[e]), lo = fminf(lo, v[e]);
    finite = fmaf(v[e], 0.0f, finite);  // NaN where one is not
  }
#pragma unroll
  for (int o = 1; o <= 2; o <<= 1) {
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
  }
  const uint32_t votes = __ballot_sync(0xffffffffu, finite != 0.0f);
  const int lane = threadIdx.x & 31;
  const bool all_finite = (votes >> (lane & ~3) & 15u) == 0;
  const float top = hi >= -lo ? hi : lo;
  __nv_bfloat16 sb = __float2bfloat16_rn(top * -0.125f);
  if (!all_finite) sb = __ushort_as_bfloat16(0x7fc0);
  const float s = __bfloat162float(sb);
  uint32_t run[2] = {0x8888u, 0x8888u};  // the codes of four dims each
  if (all_finite && s != 0.0f) codes<sizeof(T) == 2>(v, s, run);
  const uint32_t other0 = __shfl_xor_sync(0xffffffffu, run[0], 4), other1 = __shfl_xor_sync(0xffffffffu, run[1], 4);
  if (!fits) return;
  const int page = slot >> p.c.log_page, place = slot & (p.c.page - 1);
  const int64_t at = ((int64_t)page * p.c.Hkv + h) * p.c.page + place;
  uint32_t* words = reinterpret_cast<uint32_t*>(p.c.q[kv] + at * (D / 2));
  const int block = part / 8, l = part % 8;
  if (D == 96 && block == 0) {  // its eight lanes may lie in two warps: half words
    uint16_t* halves = reinterpret_cast<uint16_t*>(words) + l % 4 * 4 + l / 4;
    halves[0] = (uint16_t)run[0], halves[2] = (uint16_t)run[1];
  } else if (block * 64 + 64 <= D) {
    if (l < 4)
      *reinterpret_cast<uint2*>(words + block * 8 + l * 2) = make_uint2(run[0] | other0 << 16, run[1] | other1 << 16);
  } else {
    words[block * 8 + l] = run[0] | run[1] << 16;
  }
  if (part % 4 == 0) p.c.scale[kv][at * (D / kGroup) + part / 4] = __bfloat16_as_ushort(sb);
}

struct Read {
  Cache c;
  void* out[2];
  const int32_t *table, *lens;
  int B, M;
  int* err;
};

// Eight dims a thread, in the output's order; blockIdx.y keys or values, blockIdx.z the entry.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) read_kernel(const __grid_constant__ Read p) {
  pdl_wait();
  pdl_trigger();
  constexpr uint32_t lanes = D / 8;
  const int kv = blockIdx.y;
  const int64_t b = blockIdx.z;
  const int T_all = p.M << p.c.log_page;
  const int n = p.lens ? min(max(p.lens[b], 0), T_all) : T_all;
  const uint32_t total = lanes * p.c.Hkv * (uint32_t)T_all;
  T* out = static_cast<T*>(p.out[kv]) + b * (int64_t)total * 8;
  for (uint32_t i = blockIdx.x * kThreads + threadIdx.x; i < total; i += gridDim.x * kThreads) {
    const uint32_t row = i / lanes, part = i % lanes, t = row / (uint32_t)p.c.Hkv, h = row - t * (uint32_t)p.c.Hkv;
    float v[8] = {};
    if ((int)t < n) {
      const int page = p.table[b * p.M + (t >> p.c.log_page)];
      if ((unsigned)page < (unsigned)p.c.pages) {
        const int64_t at = ((int64_t)page * p.c.Hkv + h) * p.c.page + (t & (p.c.page - 1));
        const uint32_t* words = reinterpret_cast<const uint32_t*>(p.c.q[kv] + at * (D / 2));
        const uint32_t block = part / 8, l = part % 8;
        uint32_t codes;  // of the eight dims, ascending
        if (block * 64 + 64 <= D) {
          const uint2 w = *reinterpret_cast<const uint2*>(words + block * 8 + l % 4 * 2);
          codes = __byte_perm(w.x, w.y, l < 4 ? 0x5410 : 0x7632);
        } else {
          codes = words[block * 8 + l];
        }
        const float s = __uint_as_float((uint32_t)p.c.scale[kv][at * (D / kGroup) + part / 4] << 16);
#pragma unroll
        for (int e = 0; e < 8; ++e)  // 2^23 + code, less 2^23 + 8
          v[e] = s * (__uint_as_float(0x4b000000u | (codes >> (4 * e) & 15u)) - 8388616.0f);
      } else {
        record_error(p.err, HCLSM_ERR_SHAPE);
      }
    }
    store8(out + (int64_t)i * 8, v);
  }
}

template <typename T> int launch_write(const Write& p, dim3 g, cudaStream_t st) {
  switch (p.c.D) {
    case 32: return launch_pdl(write_kernel<T, 32>, g, kThreads, 0, st, p);
    case 64: return launch_pdl(write_kernel<T, 64>, g, kThreads, 0, st, p);
    case 96: return launch_pdl(write_kernel<T, 96>, g, kThreads, 0, st, p);
    default: return launch_pdl(write_kernel<T, 128>, g, kThreads, 0, st, p);
  }
}
template <typename T> int launch_read(const Read& p, dim3 g, cudaStream_t st) {
  switch (p.c.D) {
    case 32: return launch_pdl(read_kernel<T, 32>, g, kThreads, 0, st, p);
    case 64: return launch_pdl(read_kernel<T, 64>, g, kThreads, 0, st, p);
    case 96: return launch_pdl(read_kernel<T, 96>, g, kThreads, 0, st, p);
    default: return launch_pdl(read_kernel<T, 128>, g, kThreads, 0, st, p);
  }
}

bool al16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

int check(const hclsm_kv4_cache* c) {
  if (!c) return HCLSM_ERR_NULL;
  if (c->dtype != HCLSM_F32 && c->dtype != HCLSM_BF16) return HCLSM_ERR_DTYPE;
  if (c->pages < 0 || c->Hkv < 1) return HCLSM_ERR_SHAPE;
  if (c->D != 32 && c->D != 64 && c->D != 96 && c->D != 128) return HCLSM_ERR_SHAPE;
  if (c->page != 16 && c->page != 32 && c->page != 64 && c->page != 128) return HCLSM_ERR_SHAPE;
  if ((int64_t)c->pages * c->page > 0x7fffffff) return HCLSM_ERR_SHAPE;
  if (c->pages == 0) return HCLSM_OK;
  if (!c->k || !c->v || !c->k_scale || !c->v_scale) return HCLSM_ERR_NULL;
  if (!al16(c->k) || !al16(c->v) || !al16(c->k_scale) || !al16(c->v_scale)) return HCLSM_ERR_ALIGN;
  return HCLSM_OK;
}

bool row16(const xattn::View& v, int dtype) {
  const int e = dtype == HCLSM_F32 ? 4 : 2;
  return al16(v.p) && v.sb * e % 16 == 0 && v.st * e % 16 == 0 && v.sh * e % 16 == 0;
}

int check_table(const hclsm_kv4_cache* c, const int32_t* table, int B, int M) {
  if (B < 0 || M < 0 || (int64_t)M * c->page > 0x7fffffff) return HCLSM_ERR_SHAPE;
  return (int64_t)B * M > 0 && !table ? HCLSM_ERR_NULL : HCLSM_OK;
}

Attn attn_params(const hclsm_kv4_cache* c, int B, int M, int Lq, int H) {
  Attn p = {};
  p.c = cache(c);
  p.B = B, p.M = M, p.Lq = Lq, p.H = H;
  return p;
}

}  // namespace kv4
}  // namespace hclsm

using namespace hclsm;

extern "C" int hclsm_kv4_write(const hclsm_kv4_cache* c, const hclsm_view* k, const hclsm_view* v,
                               const int32_t* slots, int32_t B, int32_t n, void* stream) {
  if (const int rc = kv4::check(c)) return rc;
  if (B < 0 || n < 0) return HCLSM_ERR_SHAPE;
  if ((int64_t)B * n == 0) return HCLSM_OK;
  if (!k || !v || !k->p || !v->p || !slots) return HCLSM_ERR_NULL;
  kv4::Write p = {};
  p.c = kv4::cache(c);
  p.x[0] = xattn::view(*k, B, n, c->Hkv), p.x[1] = xattn::view(*v, B, n, c->Hkv);
  if (!kv4::row16(p.x[0], c->dtype) || !kv4::row16(p.x[1], c->dtype)) return HCLSM_ERR_ALIGN;
  const int64_t total = (int64_t)B * n * c->Hkv * (c->D / 8), grid = (total + kv4::kThreads - 1) / kv4::kThreads;
  if (total > 0x7fffffff) return HCLSM_ERR_SHAPE;
  p.slots = slots, p.n = n, p.total = (uint32_t)total, p.err = device_err_ptr();
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 g((unsigned)grid, 2);
  return c->dtype == HCLSM_F32 ? kv4::launch_write<float>(p, g, st) : kv4::launch_write<__nv_bfloat16>(p, g, st);
}

extern "C" int hclsm_kv4_read(const hclsm_kv4_cache* c, const int32_t* table, int32_t B, int32_t M, void* k, void* v,
                              const int32_t* lens, void* stream) {
  if (const int rc = kv4::check(c)) return rc;
  if (const int rc = kv4::check_table(c, table, B, M)) return rc;
  if ((int64_t)B * M == 0) return HCLSM_OK;
  if (!k || !v) return HCLSM_ERR_NULL;
  if (!kv4::al16(k) || !kv4::al16(v)) return HCLSM_ERR_ALIGN;
  kv4::Read p = {};
  p.c = kv4::cache(c);
  p.out[0] = k, p.out[1] = v, p.table = table, p.lens = lens, p.B = B, p.M = M, p.err = device_err_ptr();
  const int64_t total = (int64_t)M * c->page * c->Hkv * (c->D / 8);
  if (total > 0x7fffffff || B > 65535) return HCLSM_ERR_SHAPE;
  const int64_t blocks = (total + kv4::kThreads - 1) / kv4::kThreads, most = (int64_t)num_sms() * 16 / B + 1;
  const dim3 g((unsigned)(blocks < most ? blocks : most), 2, (unsigned)B);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return c->dtype == HCLSM_F32 ? kv4::launch_read<float>(p, g, st) : kv4::launch_read<__nv_bfloat16>(p, g, st);
}

extern "C" size_t hclsm_kv4_attn_workspace_size(const hclsm_kv4_cache* c, int32_t B, int32_t M, int32_t Lq,
                                                int32_t H) {
  if (kv4::check(c) || B < 0 || M < 0 || Lq < 0 || H < 1 || H % c->Hkv) return 0;
  return kv4::attn_workspace(kv4::attn_params(c, B, M, Lq, H), c->dtype);
}

extern "C" int hclsm_kv4_attn(const hclsm_kv4_cache* c, const int32_t* table, int32_t B, int32_t M,
                              const hclsm_view* q, void* o, const int32_t* lens, int32_t Lq, int32_t H, float scale,
                              void* ws, size_t ws_bytes, void* stream) {
  if (const int rc = kv4::check(c)) return rc;
  if (const int rc = kv4::check_table(c, table, B, M)) return rc;
  if (Lq < 0 || H < 1 || H % c->Hkv || !(scale > 0.0f) || scale > 3.0e38f) return HCLSM_ERR_SHAPE;
  if ((int64_t)B * Lq == 0) return HCLSM_OK;
  if (!q || !q->p || !o) return HCLSM_ERR_NULL;
  kv4::Attn p = kv4::attn_params(c, B, M, Lq, H);
  p.q = xattn::view(*q, B, Lq, H);
  if (!kv4::row16(p.q, c->dtype) || !kv4::al16(o)) return HCLSM_ERR_ALIGN;
  p.o = o, p.table = table, p.lens = lens, p.c2 = scale * kLog2e, p.err = device_err_ptr();
  const size_t need = kv4::attn_workspace(p, c->dtype);
  if (ws_bytes < need || (need && !ws)) return HCLSM_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(ws) % 16) return HCLSM_ERR_ALIGN;
  return kv4::attn(p, c->dtype, ws, static_cast<cudaStream_t>(stream));
}
