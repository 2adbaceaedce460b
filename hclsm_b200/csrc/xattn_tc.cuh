// What the bf16 cross-attention kernels on the tensor cores share: the key mask as
// bits, packed fp32 arithmetic, tensor maps.
#pragma once
#include <cuda.h>

#include <mutex>

#include "tcgen05.cuh"
#include "xattn.cuh"

namespace hclsm {
namespace xattn {

using namespace ::hclsm::tc;

constexpr int kTile = 128;            // query rows and keys of a forward tile
constexpr uint32_t kRowBytes = 128;   // a 64-dim bf16 row of a swizzled block

struct TcParams {
  Params x;
  const uint32_t* words;  // (B, word_sb) bits of the key mask, or null
  int word_sb;
  int qtiles;  // of QT * 128 rows
};

// The allowed keys of [k0, k0 + 128) as bits.
__device__ __forceinline__ uint4 key_bits(const TcParams& p, int64_t b, int n, int k0) {
  auto below = [&](int base) {
    const int left = n - base;
    return left >= 32 ? 0xffffffffu : left <= 0 ? 0u : (1u << left) - 1u;
  };
  uint4 r = make_uint4(below(k0), below(k0 + 32), below(k0 + 64), below(k0 + 96));
  if (p.words) {
    const uint4 w = *reinterpret_cast<const uint4*>(p.words + b * p.word_sb + k0 / 32);
    r.x &= w.x, r.y &= w.y, r.z &= w.z, r.w &= w.w;
  }
  return r;
}
__device__ __forceinline__ bool all_bits(const uint4& w) { return (w.x & w.y & w.z & w.w) == 0xffffffffu; }

// Zero the rows of a staged tile whose bit is off (a whole warp): an operand that
// may be NaN or stale memory must not meet a zero weight.
template <int DP, int ROWS>
__device__ __forceinline__ void zero_rows(unsigned char* tile, const uint4& w, int lane) {
  const uint32_t word[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < ROWS / 32; ++i)
    if (!(word[i] >> lane & 1u)) {
#pragma unroll
      for (int kb = 0; kb < DP / 64; ++kb) {
        uint4* row = reinterpret_cast<uint4*>(tile + ((size_t)kb * ROWS + i * 32 + lane) * kRowBytes);
#pragma unroll
        for (int c = 0; c < 8; ++c) row[c] = make_uint4(0, 0, 0, 0);
      }
    }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncwarp();
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
// 2^x of two values at most 2^8 on the FMA pipe: x = n + f with n the nearest integer
// (Cody and Waite's reduction by adding 1.5 * 2^23), 2^f by a cubic fitted here for the
// least largest relative error on [-1/2, 1/2] (7.5e-5, a fiftieth of the bf16 rounding
// that follows), 2^n from n's bits.  NaN stays NaN; below 2^-126 the result is 0.
__device__ __forceinline__ float2 ex2_fma(float2 x) {
  x.x = max_nan(x.x, -127.0f), x.y = max_nan(x.y, -127.0f);
  const float2 t = add2(x, make_float2(12582912.0f, 12582912.0f));
  const float2 n = add2(t, make_float2(-12582912.0f, -12582912.0f));
  const float2 f = fma2(n, make_float2(-1.0f, -1.0f), x);
  float2 p = fma2(f, make_float2(0.05517167f, 0.05517167f), make_float2(0.24261113f, 0.24261113f));
  p = fma2(p, f, make_float2(0.69326097f, 0.69326097f));
  p = fma2(p, f, make_float2(0.99992806f, 0.99992806f));
  return mul2(p, make_float2(__uint_as_float((__float_as_uint(t.x) << 23) + 0x3f800000u),
                             __uint_as_float((__float_as_uint(t.y) << 23) + 0x3f800000u)));
}

// ---- host ----------------------------------------------------------------------------------
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(p);
  });
  return fn;
}

// (D, L, H, B) bf16, box (64, rows, 1, 1), 128-byte swizzle, zeros outside.
inline bool make_map(CUtensorMap* m, const View& v, int D, int L, int H, int B, int rows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)L, (cuuint64_t)H, (cuuint64_t)B};
  cuuint64_t strides[3] = {(cuuint64_t)v.st * 2, (cuuint64_t)v.sh * 2, (cuuint64_t)v.sb * 2};
  for (int i = 0; i < 3; ++i)
    if (dims[i + 1] == 1) strides[i] = (cuuint64_t)((D + 7) / 8 * 16);  // never stepped over
  const cuuint32_t box[4] = {64, (cuuint32_t)rows, 1, 1};
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(v.p), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// What a tensor map can describe: 16-byte aligned rows, positive strides.
inline bool mappable(const View& v, int L, int H, int B) {
  auto ok = [](int n, int64_t s) { return n == 1 || (s > 0 && s % 8 == 0 && s < ((int64_t)1 << 38)); };
  return reinterpret_cast<uintptr_t>(v.p) % 16 == 0 && ok(L, v.st) && ok(H, v.sh) && ok(B, v.sb);
}

inline int word_stride(const Params& p) { return (p.Lk + kTile - 1) / kTile * (kTile / 32); }

// The mask's bits into ws (tc_workspace bytes) and t (xattn_tc.cu).
int make_bits(TcParams& t, void* ws, cudaStream_t st);

}  // namespace xattn
}  // namespace hclsm
