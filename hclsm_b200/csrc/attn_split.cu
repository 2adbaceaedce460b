// Attention of few query rows over long keys, the keys split over thread
// blocks: the single-token form of the cross attention (states in fp32 or
// bf16) and the attention over the 8-bit state cache.
//
// The rows that share a key head (tokens x query heads of the group) form the
// M = 16 side of mma.sync m16n8k16 products; a warp takes 16 keys a step:
//   S = Q K^T  ->  running max / sum  ->  P (fp32 accumulators become the A
//   fragments of the next product in place)  ->  O += P V.
// A contraction's index can run in any order, so fragments come straight from
// global memory with 16-byte loads and no shared memory: for S a lane's four k
// slots are four consecutive dims of its key's row; for P V a lane holds
// consecutive dims of the four keys whose scores it has.
// 8-bit integers become fp16 two at a time: 0x6400 | (x + 128) is 1152 + x.  For K
// the 1152 stays in: S is off by 1152 times the row's sum of q, one subtraction a
// score.  For V it is taken off (the sum over a long history would lose the
// difference).  For fp16's range queries are scaled by a power of two to a largest value
// below 1 (exact, but for values 2^-14 of the largest and below, which lose what is below
// 2^-24 of it: a query's channel 2^12 times its others whose keys are nearly zero takes the output from 0.16 to 0.22 %,
// one of 2^14 times to 0.6 %; bf16 there is exact and costs 18 %, 542 us against 458) and weights to at most 2^12;
// fp16's 11 bits round them less than bf16's 8.
// The scale of a block of keys multiplies its scores (K); that of its values, over the largest of weight times scale so
// far, its weights (V).
// fp32 operands are split into three bf16 pieces (8 bits each) and the products
// of pieces whose order is at most 2 are summed: fp32 accuracy.
// Bound: HBM (each key and value byte is read once); splits and warps are merged
// in a fixed order.  One query over 8 x 16384 ragged bf16 states, 16 heads over 4 of
// 128: 50 us (floor 31); over 16 x 65536 cached states, 32 heads over 8 of 128: 459 us,
// 4.7 TB/s, and 355 us, 4.4 TB/s, where the lengths are ragged (0.72 of the states).  43 % of the
// issue slots are taken, so loads in flight are the bound: 12 warps an SM, a step each in
// registers.  Three blocks an SM: four spill (415 us against 380); four waves of blocks: eight are slower (480 against
// 450).
#include <cuda_fp16.h>

#include <type_traits>

#include "xattn.cuh"

namespace hclsm {
namespace split {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kRows = 16;
constexpr int kWaves = 4, kMinKeys = 1024;

struct Params {
  xattn::Params x;  // q, o, lse2, lens, mask, sizes; k and v where the states are dense
  const int8_t *k8, *v8;      // (B, Hkv, T, D)
  const float *ks, *vs;       // (B, Hkv, T / block)
  const void *kt, *vt;        // (B, Hkv, block, D), the last incomplete block
  int T, block;
  int splits, rtiles;
  float* part_o;   // (B * Hkv * rtiles, splits, 16, D)
  float2* part_ml; // (B * Hkv * rtiles, splits, 16): max, sum
};

template <bool F16>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (F16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
        "%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, "
        "%2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// The N leading bf16 pieces of two fp32 values, packed.
template <int N>
__device__ __forceinline__ void pieces(float lo, float hi, uint32_t (&out)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    out[i] = pack(lo, hi);
    lo -= __uint_as_float(out[i] << 16);
    hi -= __uint_as_float(out[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// Two signed bytes (bits 0-7 and 16-23; the others are ignored): 1152 + x as packed fp16, and x as packed bf16
// (0x4300 | low 7 bits is 128 + those bits, 0x4300 | sign 128, or 256 for a negative value).
__device__ __forceinline__ uint32_t bytes_f16(uint32_t t) { return (t & 0x00ff00ffu) ^ 0x64806480u; }
__device__ __forceinline__ uint32_t minus1152(uint32_t t) {
  const uint32_t k = 0x64806480u;
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&t), *reinterpret_cast<const __half2*>(&k));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t bytes_bf16(uint32_t t) {
  const uint32_t m = (t & 0x007f007fu) | 0x43004300u, s = (t & 0x00800080u) | 0x43004300u;
  const __nv_bfloat162 r =
      __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&m), *reinterpret_cast<const __nv_bfloat162*>(&s));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// How one lane reads rows of D elements of type E: K as D / 4 elements (a quad
// shares a row), V as D / 8 elements (eight lanes share a row) in runs of CV
// consecutive dims.  CV fixes which dims an accumulator tile holds, so storage
// types that meet in one accumulator use the same.
constexpr int load_bytes(int bytes) { return bytes % 16 == 0 ? 16 : bytes % 8 == 0 ? 8 : 4; }

template <typename E, int D, int CV>
struct Rows {
  static constexpr int kES = (int)sizeof(E);
  static constexpr int kPieces = kES == 4 ? 3 : 1;
  static constexpr int kKB = D / 4 * kES, kVB = D / 8 * kES;  // bytes a lane reads of a row
  static constexpr int kKC = load_bytes(kKB);                 // bytes of one load
  static constexpr int kVC = load_bytes(CV * kES);
  static constexpr int kKW = kKB / 4, kVW = kVB / 4;          // words
  static constexpr int kCK = kKC / kES;                       // elements of one load of K

  template <int CB>
  static __device__ __forceinline__ void load(const char* p, uint32_t* w) {
    if constexpr (CB == 16) {
      const uint4 r = __ldcs(reinterpret_cast<const uint4*>(p));
      w[0] = r.x, w[1] = r.y, w[2] = r.z, w[3] = r.w;
    } else if constexpr (CB == 8) {
      const uint2 r = __ldcs(reinterpret_cast<const uint2*>(p));
      w[0] = r.x, w[1] = r.y;
    } else {
      w[0] = __ldcs(reinterpret_cast<const uint32_t*>(p));
    }
  }
  // row: address of the key's first element
  static __device__ __forceinline__ void load_k(const char* row, int c, uint32_t (&w)[kKW]) {
#pragma unroll
    for (int i = 0; i < kKB / kKC; ++i) load<kKC>(row + (i * 4 + c) * kKC, w + i * (kKC / 4));
  }
  static __device__ __forceinline__ void load_v(const char* row, int g, uint32_t (&w)[kVW]) {
#pragma unroll
    for (int i = 0; i < D / 8 / CV; ++i)
#pragma unroll
      for (int k = 0; k < CV * kES / kVC; ++k)
        load<kVC>(row + (i * 8 + g) * CV * kES + k * kVC, w + (i * CV * kES + k * kVC) / 4);
  }
  // the dim of lane quad-index c's element 0..3 of k step s
  static __device__ __forceinline__ int k_dim(int s, int c) {
    return s / (kCK / 4) * 4 * kCK + c * kCK + s % (kCK / 4) * 4;
  }
  // the dim of lane group g's element j
  static __device__ __forceinline__ int v_dim(int j, int g) { return j / CV * 8 * CV + g * CV + j % CV; }

  // B fragments of k step s (F16: 1152 + x)
  template <bool F16>
  static __device__ __forceinline__ void k_frag(const uint32_t (&w)[kKW], int s, uint32_t (&b0)[kPieces],
                                                uint32_t (&b1)[kPieces]) {
    if constexpr (kES == 1) {
      if constexpr (F16) {
        const uint32_t u = w[s] ^ 0x80808080u;
        b0[0] = __byte_perm(u, 0x64646464u, 0x4140), b1[0] = __byte_perm(u, 0x64646464u, 0x4342);
      } else {
        b0[0] = bytes_bf16(__byte_perm(w[s], 0, 0x0100)), b1[0] = bytes_bf16(__byte_perm(w[s], 0, 0x0302));
      }
    } else if constexpr (kES == 2) {
      b0[0] = w[2 * s], b1[0] = w[2 * s + 1];
    } else {
      pieces<3>(__uint_as_float(w[4 * s]), __uint_as_float(w[4 * s + 1]), b0);
      pieces<3>(__uint_as_float(w[4 * s + 2]), __uint_as_float(w[4 * s + 3]), b1);
    }
  }
  // B fragments of n tile j from the rows of the lane's four keys
  template <bool F16>
  static __device__ __forceinline__ void v_frag(const uint32_t (&w)[4][kVW], int j, uint32_t (&b0)[kPieces],
                                                uint32_t (&b1)[kPieces]) {
    if constexpr (kES == 1) {
      const uint32_t sel = (j & 3) | ((4 + (j & 3)) << 8);  // byte j of the first word, of the second at bit 16
      const uint32_t t0 = __byte_perm(w[0][j / 4], w[1][j / 4], sel), t1 = __byte_perm(w[2][j / 4], w[3][j / 4], sel);
      b0[0] = F16 ? minus1152(bytes_f16(t0)) : bytes_bf16(t0);
      b1[0] = F16 ? minus1152(bytes_f16(t1)) : bytes_bf16(t1);
    } else if constexpr (kES == 2) {
      const uint32_t sel = j & 1 ? 0x7632 : 0x5410;
      b0[0] = __byte_perm(w[0][j / 2], w[1][j / 2], sel);
      b1[0] = __byte_perm(w[2][j / 2], w[3][j / 2], sel);
    } else {
      pieces<3>(__uint_as_float(w[0][j]), __uint_as_float(w[1][j]), b0);
      pieces<3>(__uint_as_float(w[2][j]), __uint_as_float(w[3][j]), b1);
    }
  }
};

// A warp's running state over its keys.
template <int D>
struct State {
  float o[D / 8][4];
  float m[2], l[2];
};

// The 8-bit blocks' O is held over v, times 2^12: a row's largest product so far of a step's largest weight (relative
// to the row's maximum score, 2^-115 at least, so that no factor overflows) and its block's value scale; at least
// 2^-110, where the smallest step of an fp16 weight is below bf16's smallest number.
constexpr float kLeast = 7.703719777548943e-34f, kFaint = 2.407412430484045e-35f;
struct Ref {
  float v[2] = {kLeast, kLeast}, inv[2] = {4096.0f / kLeast, 4096.0f / kLeast};  // 2^12 / v
};

// Blocks an SM: what the registers of a row's accumulators and one step's keys and values leave room for.
template <typename T, int D> constexpr int kPerSm = sizeof(T) == 4 ? (D <= 64 ? 3 : 2) : (D <= 64 ? 4 : 3);

// The A fragments of all k steps and pieces, as each lane reads them: [k step][piece][lane][2 NR words].
template <int D, int NQ, int NR> constexpr int frag_words() { return D / 16 * NQ * 32 * 2 * NR; }

// Packs them from fp32 queries [16][D + 4] (rows past the end are zeros); warps take k steps in turn.
template <int D, int NQ, int NR, bool F16, typename R>
__device__ __forceinline__ void pack_q(uint32_t* qf, const float* sq, const float* inv, int warp, int g, int c) {
  for (int s = warp; s < D / 16; s += kWarps) {
    const int d = R::k_dim(s, c);
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      const float4 x = *reinterpret_cast<const float4*>(sq + (g + 8 * r) * (D + 4) + d);
      uint32_t lo[NQ], hi[NQ];
      if constexpr (F16) {
        const float f = inv[g + 8 * r];
        lo[0] = pack_f16(x.x * f, x.y * f), hi[0] = pack_f16(x.z * f, x.w * f);
      } else {
        pieces<NQ>(x.x, x.y, lo);
        pieces<NQ>(x.z, x.w, hi);
      }
#pragma unroll
      for (int i = 0; i < NQ; ++i) {  // words: (row g, low k), (row g, high k), then row g + 8
        uint32_t* w = qf + ((s * NQ + i) * 32 + g * 4 + c) * 2 * NR + 2 * r;
        w[0] = lo[i], w[1] = hi[i];
      }
    }
  }
}
template <int NR>
__device__ __forceinline__ void load_a(const uint32_t* w, uint32_t (&a)[4]) {
  if constexpr (NR == 1) {
    const uint2 v = *reinterpret_cast<const uint2*>(w);
    a[0] = v.x, a[1] = 0, a[2] = v.y, a[3] = 0;
  } else {
    const uint4 v = *reinterpret_cast<const uint4*>(w);
    a[0] = v.x, a[1] = v.z, a[2] = v.y, a[3] = v.w;
  }
}

// NR 1: at most 8 rows, so rows g + 8 are padding that takes no softmax.
// Steps first, first + stride, ... below last of 16 keys each.  addr_k / addr_v
// (key) give a row's address; ok(key) says whether the key is allowed (false
// past the end); nk > 0 keys have memory; all_ok(step) skips the per-key checks.
// fs, off: factor and offset of rows g and g + 8's raw scores.
template <typename E, int D, int CV, int NQ, int NR, bool F16, typename AddrK, typename AddrV, typename Ok,
          typename AllOk, typename Scale>
__device__ __forceinline__ void sweep(State<D>& st, const uint32_t* qf, const float (&fs)[2], const float (&off)[2],
                                      Ref& ref, int first, int last, int stride, int nk,
                                      AddrK addr_k, AddrV addr_v, Ok ok, AllOk all_ok, Scale scale) {
  using R = Rows<E, D, CV>;
  // fp32: a product is formed from zero and added here, because the tensor core's own
  // sum over steps is not rounded to nearest (1.2e-6 instead of 5e-7 off at 5000 keys)
  constexpr bool kFull = NQ == 3;
  constexpr int NK = R::kPieces, kOrder = (NQ > NK ? NQ : NK) - 1;
  const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  if (first >= last) return;
  uint32_t kr[2][R::kKW], vr[4][R::kVW];
  auto fetch_k = [&](int step) {
#pragma unroll
    for (int t = 0; t < 2; ++t) R::load_k(addr_k(min(step * 16 + t * 8 + g, nk - 1)), c, kr[t]);
  };
  auto fetch_v = [&](int step) {
#pragma unroll
    for (int t = 0; t < 4; ++t) R::load_v(addr_v(min(step * 16 + (t >> 1) * 8 + 2 * c + (t & 1), nk - 1)), g, vr[t]);
  };
  float2 sc = scale(first);
  fetch_k(first);
  fetch_v(first);
  for (int step = first; step < last; step += stride) {
    const int next = step + stride < last ? step + stride : step;
    if (const int far = step + 2 * stride; far < last) {  // the step after the next from DRAM to L2
      constexpr int kLines = D * R::kES >= 128 ? D * R::kES / 128 : 1;  // of a row
#pragma unroll
      for (int at = lane; at < 16 * kLines; at += 32) {
        const int j = min(far * 16 + at / kLines, nk - 1);
        asm volatile("prefetch.global.L2 [%0];" ::"l"(addr_k(j) + at % kLines * 128));
        asm volatile("prefetch.global.L2 [%0];" ::"l"(addr_v(j) + at % kLines * 128));
      }
    }
    float s[2][4] = {};
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      uint32_t a[NQ][4];
#pragma unroll
      for (int i = 0; i < NQ; ++i) load_a<NR>(qf + ((ks * NQ + i) * 32 + lane) * 2 * NR, a[i]);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        uint32_t b0[NK], b1[NK];
        R::template k_frag<F16>(kr[t], ks, b0, b1);
        float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = NQ - 1; i >= 0; --i)
#pragma unroll
          for (int j = NK - 1; j >= 0; --j)
            if (i + j <= kOrder) mma<F16>(kFull ? part : s[t], a[i], b0[j], b1[j]);
        if constexpr (kFull) {
#pragma unroll
          for (int e = 0; e < 2 * NR; ++e) s[t][e] += part[e];
        }
      }
    }
    const float2 cur = sc;
    sc = scale(next);
    fetch_k(next);
    // ---- running max and sum; a lane's scores: rows g, g + 8, keys 8 t + 2 c, + 1
    const bool all = all_ok(step);
    bool good[4] = {true, true, true, true};
    if (!all) {
#pragma unroll
      for (int t = 0; t < 4; ++t) good[t] = ok(step * 16 + (t >> 1) * 8 + 2 * c + (t & 1));
    }
    const float f[2] = {fs[0] * cur.x, fs[1] * cur.x};
    float mx[2] = {-INFINITY, -INFINITY};  // of this step alone where F16
    if constexpr (!F16) mx[0] = st.m[0], mx[1] = st.m[1];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < 2 * NR; ++e) {
        if constexpr (F16) s[t][e] -= off[e >> 1];
        s[t][e] = good[2 * t + (e & 1)] ? s[t][e] * f[e >> 1] : -INFINITY;
        mx[e >> 1] = fmaxf(mx[e >> 1], s[t][e]);
      }
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
      mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
    }
    float pv[2] = {cur.y, cur.y};
    if constexpr (F16) {
      // Weights are at most 2^12 through the largest weight times scale, not the largest scale: a block of large values
      // that no weight falls on would take the others' weights below fp16's range.
      float top[2];
      bool more = false;
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        const float m = fmaxf(st.m[r], mx[r]);
        top[r] = cur.y * fmaxf(ex2(mx[r] - m), kFaint);  // NaN where both are -inf: kFaint
        mx[r] = m;
        more |= m != st.m[r] || top[r] > ref.v[r];
      }
      if (__any_sync(0xffffffffu, more)) {
#pragma unroll
        for (int r = 0; r < NR; ++r) {
          const float w = mx[r] == -INFINITY ? 1.0f : ex2(st.m[r] - mx[r]);
          st.m[r] = mx[r];
          st.l[r] *= w;
          const float old = ref.v[r] * w;  // a new maximum lowers O through it
          ref.v[r] = fmaxf(fmaxf(old, top[r]), kLeast);
          ref.inv[r] = 4096.0f / ref.v[r];
          if (ref.v[r] != old) {
            const float f = old / ref.v[r];
#pragma unroll
            for (int j = 0; j < D / 8; ++j) st.o[j][2 * r] *= f, st.o[j][2 * r + 1] *= f;
          }
        }
      }
#pragma unroll
      for (int r = 0; r < NR; ++r) pv[r] *= ref.inv[r];  // a scale of 0 or NaN stays
    } else if (__any_sync(0xffffffffu, mx[0] != st.m[0] || mx[1] != st.m[1])) {
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        const float w = mx[r] == -INFINITY ? 1.0f : ex2(st.m[r] - mx[r]);
        st.m[r] = mx[r];
        st.l[r] *= w;
#pragma unroll
        for (int j = 0; j < D / 8; ++j) st.o[j][2 * r] *= w, st.o[j][2 * r + 1] *= w;
      }
    }
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (e >= 2 * NR) {
          s[t][e] = 0.0f;
          continue;
        }
        const float base = st.m[e >> 1] == -INFINITY ? 0.0f : st.m[e >> 1];
        s[t][e] = ex2(s[t][e] - base);
        st.l[e >> 1] += s[t][e];
        s[t][e] *= pv[e >> 1];
        if (!all && !good[2 * t + (e & 1)]) s[t][e] = 0.0f;
      }
    uint32_t pa[NQ][4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float lo = s[k >> 1][2 * (k & 1)], hi = s[k >> 1][2 * (k & 1) + 1];
      uint32_t t[NQ];
      if constexpr (F16) t[0] = pack_f16(lo, hi);
      else pieces<NQ>(lo, hi, t);
#pragma unroll
      for (int i = 0; i < NQ; ++i) pa[i][k] = t[i];
    }
    if (!all) {  // what is not allowed is no operand: 0 * NaN is NaN
#pragma unroll
      for (int t = 0; t < 4; ++t)
        if (!good[t]) {
#pragma unroll
          for (int w = 0; w < R::kVW; ++w) vr[t][w] = 0;
        }
    }
#pragma unroll
    for (int j = 0; j < D / 8; ++j) {
      uint32_t b0[NK], b1[NK];
      R::template v_frag<F16>(vr, j, b0, b1);
      float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int i = NQ - 1; i >= 0; --i)
#pragma unroll
        for (int k = NK - 1; k >= 0; --k)
          if (i + k <= kOrder) mma<F16>(kFull ? part : st.o[j], pa[i], b0[k], b1[k]);
      if constexpr (kFull) {
#pragma unroll
        for (int e = 0; e < 2 * NR; ++e) st.o[j][e] += part[e];
      }
    }
    fetch_v(next);
  }
}

template <typename T>
__device__ __forceinline__ void store_o(const xattn::Params& x, int64_t at, float v) {
  io<T>::st(static_cast<T*>(x.o) + at, v);
  if (sizeof(T) == 2 && x.lo) x.lo[at] = __float2bfloat16_rn(xattn::rounding(v));
}

template <typename T, int D, bool CACHE, int NR>
__global__ void __launch_bounds__(kThreads, kPerSm<T, D>) split_kernel(const __grid_constant__ Params p) {
  constexpr int NQ = sizeof(T) == 4 ? 3 : 1;
  constexpr int ES = CACHE ? 1 : (int)sizeof(T), CV = load_bytes(D / 8 * ES) / ES;
  constexpr bool F16 = CACHE && NQ == 1;
  extern __shared__ float smem[];  // [16][D + 4] queries and the A fragments, then (merge) [kWarps][16][D]
  __shared__ float s_inv[kRows], s_sum[kRows];
  __shared__ float s_m[kWarps][kRows], s_l[kWarps][kRows];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  pdl_wait();
  pdl_trigger();
  const int rt = (int)(blockIdx.x % p.rtiles);
  const int sp = (int)(blockIdx.x / p.rtiles % p.splits);
  const int64_t bh = blockIdx.x / p.rtiles / p.splits;
  const int64_t b = bh / p.x.Hkv;
  const int hk = (int)(bh % p.x.Hkv);
  const int G = p.x.H / p.x.Hkv;
  const int rows = p.x.Lq * G;  // row r: token r / G, head hk * G + r % G
  const int n = p.x.lens ? min(max(p.x.lens[b], 0), CACHE ? p.T : p.x.Lk) : (CACHE ? p.T : p.x.Lk);
  float* sq = smem;
  for (int i = threadIdx.x; i < kRows * D; i += kThreads) {
    const int r = rt * kRows + i / D, d = i % D;
    float v = 0.0f;
    if (r < rows)
      v = io<T>::ld(static_cast<const T*>(p.x.q.p) + b * p.x.q.sb + (int64_t)(r / G) * p.x.q.st +
                    (int64_t)(hk * G + r % G) * p.x.q.sh + d);
    sq[i / D * (D + 4) + d] = v;
  }
  __syncthreads();
  uint32_t* qf = reinterpret_cast<uint32_t*>(sq + kRows * (D + 4));  // as the sweep over dense states reads them
  uint32_t* qh = qf + frag_words<D, NQ, NR>();                       // fp16, for the 8-bit blocks
  using RT = Rows<T, D, CV>;
  if constexpr (F16) {  // each row times a power of two, to a largest value in [1/2, 1), and its sum
    for (int r = warp; r < kRows; r += kWarps) {
      float m = 0.0f;
      for (int d = lane; d < D; d += 32) m = fmaxf(m, fabsf(sq[r * (D + 4) + d]));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      const int e = min(max((int)(__float_as_uint(m) >> 23) - 126, -126), 126);
      const float f = m == 0.0f ? 1.0f : __uint_as_float((uint32_t)(127 - e) << 23);
      float sum = 0.0f;
      for (int d = lane; d < D; d += 32) sum += __half2float(__float2half_rn(sq[r * (D + 4) + d] * f));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane == 0) s_inv[r] = f, s_sum[r] = sum;
    }
    __syncthreads();
    pack_q<D, 1, NR, true, Rows<int8_t, D, CV>>(qh, sq, s_inv, warp, g, c);
    pack_q<D, 1, NR, false, RT>(qf, sq, s_inv, warp, g, c);
  } else if constexpr (CACHE) {
    pack_q<D, NQ, NR, false, Rows<int8_t, D, CV>>(qh, sq, s_inv, warp, g, c);
    pack_q<D, NQ, NR, false, RT>(qf, sq, s_inv, warp, g, c);
  } else {
    pack_q<D, NQ, NR, false, RT>(qf, sq, s_inv, warp, g, c);
  }
  __syncthreads();
  State<D> st;
#pragma unroll
  for (int j = 0; j < D / 8; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) st.o[j][e] = 0.0f;
  st.m[0] = st.m[1] = -INFINITY;
  st.l[0] = st.l[1] = 0.0f;
  const float c2 = p.x.scale * kLog2e;
  const float fs[2] = {c2, c2}, off[2] = {0.0f, 0.0f};
  // this block's share of the sequence's own steps
  const int n8 = CACHE ? n / p.block * p.block : n;
  const int steps = (n8 + 15) / 16, per = (steps + p.splits - 1) / p.splits;
  const int first = min(steps, sp * per), last = min(steps, first + per);
  if constexpr (CACHE) {
    const char* k8 = reinterpret_cast<const char*>(p.k8) + bh * p.T * D;
    const char* v8 = reinterpret_cast<const char*>(p.v8) + bh * p.T * D;
    const int64_t s0 = bh * (p.T / p.block);
    const int spb = p.block / 16;
    float fs8[2] = {c2, c2}, off8[2] = {0.0f, 0.0f};
    if constexpr (F16) {
#pragma unroll
      for (int r = 0; r < 2; ++r) fs8[r] = c2 / s_inv[g + 8 * r], off8[r] = 1152.0f * s_sum[g + 8 * r];
    }
    Ref ref;
    auto scale = [&](int step) { return make_float2(p.ks[s0 + step / spb], p.vs[s0 + step / spb]); };
    auto key = [&](int j) { return k8 + (int64_t)j * D; };
    auto value = [&](int j) { return v8 + (int64_t)j * D; };
    sweep<int8_t, D, CV, NQ, NR, F16>(
        st, qh, fs8, off8, ref, first + warp, last, kWarps, n8, key, value, [](int) { return true; },
        [](int) { return true; }, scale);
    // a length inside a block: a complete one (8 bits), or the one that the tail holds (scale -1)
    const bool more = sp == p.splits - 1 && n > n8;
    const bool tail = more && p.ks[s0 + n8 / p.block] < 0.0f;
    if (more && !tail)
      sweep<int8_t, D, CV, NQ, NR, F16>(
          st, qh, fs8, off8, ref, steps + warp, (n + 15) / 16, kWarps, n, key, value, [&](int j) { return j < n; },
          [&](int step) { return step * 16 + 16 <= n; }, scale);
    if constexpr (F16) {
#pragma unroll
      for (int j = 0; j < D / 8; ++j)
#pragma unroll
        for (int e = 0; e < 2 * NR; ++e) st.o[j][e] *= ref.v[e >> 1] * (1.0f / 4096.0f);
    }
    if (tail) {
      const char* kt = reinterpret_cast<const char*>(static_cast<const T*>(p.kt) + bh * p.block * D);
      const char* vt = reinterpret_cast<const char*>(static_cast<const T*>(p.vt) + bh * p.block * D);
      const int nt = n - n8;
      sweep<T, D, CV, NQ, NR, false>(
          st, qf, fs, off, ref, warp, (nt + 15) / 16, kWarps, nt, [&](int j) { return kt + j * (int)(D * sizeof(T)); },
          [&](int j) { return vt + j * (int)(D * sizeof(T)); }, [&](int j) { return j < nt; },
          [&](int step) { return step * 16 + 16 <= nt; }, [](int) { return make_float2(1.0f, 1.0f); });
    }
  } else {
    Ref ref;
    const char* kb = reinterpret_cast<const char*>(static_cast<const T*>(p.x.k.p) + b * p.x.k.sb + hk * p.x.k.sh);
    const char* vb = reinterpret_cast<const char*>(static_cast<const T*>(p.x.v.p) + b * p.x.v.sb + hk * p.x.v.sh);
    const int64_t kst = p.x.k.st * (int64_t)sizeof(T), vst = p.x.v.st * (int64_t)sizeof(T);
    sweep<T, D, CV, NQ, NR, false>(
        st, qf, fs, off, ref, first + warp, last, kWarps, n, [&](int j) { return kb + j * kst; },
        [&](int j) { return vb + j * vst; }, [&](int j) { return xattn::key_ok(p.x, b, n, j); },
        [&](int step) { return !p.x.mask && step * 16 + 16 <= n; }, [](int) { return make_float2(1.0f, 1.0f); });
  }
  // ---- merge the warps, in order -----------------------------------------------------
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    st.l[r] += __shfl_xor_sync(0xffffffffu, st.l[r], 1);
    st.l[r] += __shfl_xor_sync(0xffffffffu, st.l[r], 2);
    if (c == 0) s_m[warp][g + 8 * r] = st.m[r], s_l[warp][g + 8 * r] = st.l[r];
  }
  __syncthreads();  // the queries are done with
  using R = Rows<T, D, CV>;
#pragma unroll
  for (int j = 0; j < D / 8; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      smem[(warp * kRows + g + 8 * (e >> 1)) * D + R::v_dim(j, 2 * c + (e & 1))] = st.o[j][e];
  __shared__ float s_w[kWarps][kRows];
  if (threadIdx.x < kRows) {
    const int r = threadIdx.x;
    float m = -INFINITY, l = 0.0f;
    for (int w = 0; w < kWarps; ++w) m = fmaxf(m, s_m[w][r]);
    for (int w = 0; w < kWarps; ++w) {
      // a part without a maximum holds zeros, or NaN that has to stay
      const float f = s_m[w][r] == -INFINITY ? 1.0f : ex2(s_m[w][r] - m);
      s_w[w][r] = f;
      l += f * s_l[w][r];
    }
    const int row = rt * kRows + r;
    if (p.splits > 1) {
      p.part_ml[((bh * p.rtiles + rt) * p.splits + sp) * kRows + r] = make_float2(m, l);
    } else {
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      for (int w = 0; w < kWarps; ++w) s_w[w][r] *= inv;
      if (p.x.lse2 && row < rows)
        p.x.lse2[(b * p.x.H + hk * G + row % G) * p.x.Lq + row / G] = l == 0.0f ? INFINITY : m + log2f(l);
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < kRows * D; i += kThreads) {
    const int r = i / D, d = i % D, row = rt * kRows + r;
    if (row >= rows) break;
    float a = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) a += s_w[w][r] * smem[(w * kRows + r) * D + d];
    if (p.splits > 1)
      p.part_o[(((bh * p.rtiles + rt) * p.splits + sp) * kRows + r) * D + d] = a;
    else
      store_o<T>(p.x, ((b * p.x.Lq + row / G) * p.x.H + hk * G + row % G) * (int64_t)D + d, a);
  }
}

// One warp a row: the splits' parts, in order.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) join_kernel(const __grid_constant__ Params p) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  const int G = p.x.H / p.x.Hkv, rows = p.x.Lq * G;
  const int64_t at = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (at >= (int64_t)p.x.B * p.x.Hkv * rows) return;
  const int64_t bh = at / rows, b = bh / p.x.Hkv;
  const int row = (int)(at % rows), h = (int)(bh % p.x.Hkv) * G + row % G;
  const int64_t part = ((bh * p.rtiles + row / kRows) * p.splits) * kRows + row % kRows;
  float m = -INFINITY;
  for (int s = lane; s < p.splits; s += 32) m = fmaxf(m, p.part_ml[part + (int64_t)s * kRows].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  float l = 0.0f, acc[D / 32] = {};
#pragma unroll 4
  for (int s = 0; s < p.splits; ++s) {
    const float2 ml = p.part_ml[part + (int64_t)s * kRows];
    const float f = ml.x == -INFINITY ? 1.0f : ex2(ml.x - m);
    l += f * ml.y;
    const float* o = p.part_o + (part + (int64_t)s * kRows) * D;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) acc[i] += f * o[lane + 32 * i];
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const int64_t out = ((b * p.x.Lq + row / G) * p.x.H + h) * (int64_t)D;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) store_o<T>(p.x, out + lane + 32 * i, acc[i] * inv);
  if (p.x.lse2 && lane == 0) p.x.lse2[(b * p.x.H + h) * p.x.Lq + row / G] = l == 0.0f ? INFINITY : m + log2f(l);
}

// Whole waves of resident blocks.  Sequences have their own lengths and a block's
// share is its own sequence's, so more waves even the blocks out, down to 1024 keys a
// block (a block writes up to 16 rows of fp32 for the join).
void plan(Params& p, int keys, int dtype) {
  const int64_t rows = (int64_t)p.x.Lq * (p.x.H / p.x.Hkv);
  p.rtiles = (int)((rows + kRows - 1) / kRows);
  const int64_t base = (int64_t)p.x.B * p.x.Hkv * p.rtiles;
  const int per_sm = dtype == HCLSM_F32 ? (p.x.D <= 64 ? 3 : 2) : (p.x.D <= 64 ? 4 : 3);
  int64_t s = 1;
  for (int waves = 1; waves <= kWaves; ++waves) {
    const int64_t n = base > 0 ? (int64_t)num_sms() * per_sm * waves / base : 1;
    if (n > 1 && (waves == 1 || keys / n >= kMinKeys)) s = n;
  }
  const int64_t most = (keys + 127) / 128;
  if (s > most) s = most;
  p.splits = s < 1 ? 1 : (int)s;
}

size_t workspace(const Params& p) {
  if (p.splits <= 1) return 0;
  const size_t n = (size_t)p.x.B * p.x.Hkv * p.rtiles * p.splits * kRows;
  return n * (p.x.D * sizeof(float) + sizeof(float2));
}

template <typename T, int D, bool CACHE>
int launch(Params& p, void* ws, cudaStream_t st) {
  const int64_t grid = (int64_t)p.x.B * p.x.Hkv * p.rtiles * p.splits;
  const int64_t rows = (int64_t)p.x.B * p.x.H * p.x.Lq;
  if (grid > 0x7fffffff || rows / kWarps > 0x7ffffff0) return HCLSM_ERR_SHAPE;
  if (p.splits > 1) {
    p.part_ml = static_cast<float2*>(ws);
    p.part_o = reinterpret_cast<float*>(p.part_ml + grid * kRows);
  }
  const bool rows1 = (int64_t)p.x.Lq * (p.x.H / p.x.Hkv) <= 8;
  constexpr int NQ = sizeof(T) == 4 ? 3 : 1;
  const size_t merge = (size_t)kWarps * kRows * D * sizeof(float);
  const size_t front = (size_t)kRows * (D + 4) * sizeof(float) +
                       (size_t)(CACHE ? 2 : 1) * 4 * (rows1 ? frag_words<D, NQ, 1>() : frag_words<D, NQ, 2>());
  const size_t smem = merge > front ? merge : front;
  auto f = rows1 ? split_kernel<T, D, CACHE, 1> : split_kernel<T, D, CACHE, 2>;
  if (!set_smem_limit(reinterpret_cast<const void*>(f), smem)) return HCLSM_ERR_LAUNCH;
  if (const int rc = launch_pdl(f, (unsigned)grid, kThreads, smem, st, p)) return rc;
  if (p.splits <= 1) return HCLSM_OK;
  return launch_pdl(join_kernel<T, D>, (unsigned)((rows + kWarps - 1) / kWarps), kThreads, 0, st, p);
}

template <bool CACHE>
int run(Params& p, int dtype, void* ws, cudaStream_t st) {
  const bool f = dtype == HCLSM_F32;
  switch (p.x.D) {
    case 32: return f ? launch<float, 32, CACHE>(p, ws, st) : launch<__nv_bfloat16, 32, CACHE>(p, ws, st);
    case 64: return f ? launch<float, 64, CACHE>(p, ws, st) : launch<__nv_bfloat16, 64, CACHE>(p, ws, st);
    case 96: return f ? launch<float, 96, CACHE>(p, ws, st) : launch<__nv_bfloat16, 96, CACHE>(p, ws, st);
    case 128: return f ? launch<float, 128, CACHE>(p, ws, st) : launch<__nv_bfloat16, 128, CACHE>(p, ws, st);
  }
  return HCLSM_ERR_UNSUPPORTED;
}

}  // namespace split

namespace xattn {
// The cross attention's forward in this form; 16-byte aligned rows of k and v, D 32, 64, 96 or 128.
size_t split_workspace(const Params& x, int dtype) {
  split::Params p = {};
  p.x = x;
  split::plan(p, x.Lk, dtype);
  return split::workspace(p);
}
int split_fwd(const Params& x, int dtype, void* ws, cudaStream_t st) {
  split::Params p = {};
  p.x = x;
  split::plan(p, x.Lk, dtype);
  return split::run<false>(p, dtype, ws, st);
}
}  // namespace xattn

namespace kv8 {
size_t attn_workspace(const hclsm_kv8_cache* c, int Lq, int H) {
  split::Params p = {};
  p.x.B = c->B, p.x.Lq = Lq, p.x.H = H, p.x.Hkv = c->Hkv, p.x.D = c->D;
  split::plan(p, c->T, c->dtype);
  return split::workspace(p);
}
int attn(const hclsm_kv8_cache* c, const hclsm_view* q, void* o, const int32_t* lens, int Lq, int H, float scale,
         void* ws, cudaStream_t st) {
  split::Params p = {};
  p.x.q = xattn::view(*q, c->B, Lq, H);
  p.x.o = o, p.x.lens = lens, p.x.scale = scale;
  p.x.B = c->B, p.x.Lq = Lq, p.x.H = H, p.x.Hkv = c->Hkv, p.x.D = c->D;
  p.k8 = c->k, p.v8 = c->v, p.ks = c->k_scale, p.vs = c->v_scale, p.kt = c->k_tail, p.vt = c->v_tail;
  p.T = c->T, p.block = c->block;
  split::plan(p, c->T, c->dtype);
  return split::run<true>(p, c->dtype, ws, st);
}
}  // namespace kv8
}  // namespace hclsm
