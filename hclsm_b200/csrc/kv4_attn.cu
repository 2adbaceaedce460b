// Attention of few query rows over the paged 4-bit state cache.
//
// The rows that share a key head (tokens x query heads of the group) are the N = 8 side of mma.sync m16n8k16
// products, so that few rows waste nothing; a warp takes 32 tokens a step and keeps its own running maximum, sum and
// output.  Each warp has a ring of stages of its own, filled by bulk copies that one elected lane asks for (a page of
// one head is contiguous): no barrier between warps until the merge.
//
// A contraction's index can run in any order, so the products take the codes as they lie: two words' halves of the same
// 32 dims (or of two tokens) side by side, four bits at a time, 0x4300 | code = 128 + code in bf16.
//   S^T = K Q^T by groups of 32 dims, each times its key's scale: the 136 = 128 + 8 in every operand is taken off by
//   starting the sum at -136 times the row's sum of q in the group (fp32 states: off every operand instead,
//   their scores would lose 5 bits).
//   O^T += V^T P^T, P times the value's scale of the group before it is rounded to bf16: the codes are exact, so a weight
//   is rounded once.  movmatrix turns the scores' fragments into P^T's.  The 136 comes off the operand (summed over a
//   history it would drown the values).
// fp32 states: queries and weights as three bf16 pieces, whose products with exact codes are summed in fp32.
// The bound is issue, above all the integer pipe that unpacks the codes (60 %; issue slots 69 %, tensor pipe 23 %, 16 warps an
// SM): one query over 16 x 65536 ragged tokens, 32 heads over 8 of 128, 224 us, 4.0 TB/s.  From 450: the rows as N = 8
// instead of M = 16 (323), one operation a pair of codes (284), scales widened to fp32 once a step and four blocks an SM of
// two stages (268), one elected lane for the copies and a uniform warp index, whose addresses then cost no vector
// instructions (232), long histories first (226), a maximum that may lag behind (224).  Not kept: shifts as the upper half of
// products (317), queries and codes as e4m3 (318; its products convert them), codes as tiny bf16 numbers, which need no shift
// but a sum of their own to take off the 8 (244), 2, 3, 5, 6 or 8 waves of blocks (237, 238, 230, 238, 250).
#include <cooperative_groups.h>

#include "kv4.cuh"
#include "tcgen05.cuh"

namespace hclsm {
namespace kv4 {

constexpr int kWarps = 4, kThreads = kWarps * 32, kUnit = 32;
constexpr int kWaves = 4, kMinKeys = 1024;

// Resident blocks a SM: what the registers of a block allow.
constexpr int blocks_per_sm(bool f32, int D, int rt) { return f32 ? (D <= 64 ? 3 : 2) : D <= 64 ? 5 - rt : 4 - (rt > 1); }
// RT: tiles of 8 rows a block.
template <typename T, int D, int RT> struct Shape {
  static constexpr bool kF32 = sizeof(T) == 4;
  static constexpr int kRows = 8 * RT;
  static constexpr int kNQ = kF32 ? 3 : 1;  // bf16 pieces of a query or weight
  static constexpr int kG = D / kGroup;
  static constexpr int kCodes = kUnit * D / 2, kScales = kUnit * D / 16;  // bytes
  static constexpr int kStage = 2 * (kCodes + kScales);
  static constexpr int kStages = D == 128 ? 2 : 3;
  static constexpr int kFrag = kF32 ? kNQ * kG * 2 * 32 * 8 * RT : 0;  // query fragments of fp32 states
  static constexpr int kMerge = kWarps * kRows * D * 4;
  static constexpr int kRing = kWarps * kStages * kStage;
  static constexpr int kWide = kWarps * 2 * kUnit * kG * 4;  // a unit's scales in fp32
  static constexpr int kBytes = (kRing > kMerge ? kRing : kMerge) + kFrag + kWide;
  static constexpr int kPerSm = blocks_per_sm(kF32, D, RT);
};

// d = a b + c: with a sum of its own, the first product of a sum needs no copy of what it starts from.
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, float c0, float c1,
                                    float c2, float c3) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, "
      "%12, %13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  mma(d, a, b0, b1, d[0], d[1], d[2], d[3]);
}
// An 8 x 8 matrix of bf16 across the warp (lane 4 g + c: row g, columns 2 c and 2 c + 1), transposed.
__device__ __forceinline__ uint32_t turned(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <int N> __device__ __forceinline__ void pieces(float lo, float hi, uint32_t (&out)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    out[i] = pack(lo, hi);
    lo -= __uint_as_float(out[i] << 16);
    hi -= __uint_as_float(out[i] & 0xffff0000u);
  }
}
// Bits 0-3 and 16-19 as packed bf16: 128 + code, and code - 8.  One three-input operation with 0x43004300 in a register
// (an instruction takes one constant).
__device__ __forceinline__ uint32_t biased(uint32_t x, uint32_t k128) {
  uint32_t y;
  asm("lop3.b32 %0, %1, 0x000f000f, %2, 0xEA;" : "=r"(y) : "r"(x), "r"(k128));
  return y;
}
__device__ __forceinline__ uint32_t centred(uint32_t x, uint32_t k128) {
  const uint32_t b = biased(x, k128), k = 0x43084308u;
  const __nv_bfloat162 r =
      __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&b), *reinterpret_cast<const __nv_bfloat162*>(&k));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// A token's scales of all groups, in fp32.
template <int G> __device__ __forceinline__ void scales(const float* at, float (&s)[G]) {
  if constexpr (G == 4) {
    const float4 w = *reinterpret_cast<const float4*>(at);
    s[0] = w.x, s[1] = w.y, s[2] = w.z, s[3] = w.w;
  } else if constexpr (G == 2) {
    const float2 w = *reinterpret_cast<const float2*>(at);
    s[0] = w.x, s[1] = w.y;
  } else {
#pragma unroll
    for (int i = 0; i < G; ++i) s[i] = at[i];
  }
}

template <typename T, int D, int RT>
__global__ void __launch_bounds__(kThreads, Shape<T, D, RT>::kPerSm) attn_kernel(const __grid_constant__ Attn p) {
  using Sh = Shape<T, D, RT>;
  constexpr int G = Sh::kG, NQ = Sh::kNQ, ST = Sh::kStages, kRows = Sh::kRows;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ uint64_t bars[kWarps * ST];
  __shared__ int s_len[kThreads], s_entry;
  __shared__ float s_m[kWarps][kRows], s_l[kWarps][kRows], s_w[kWarps][kRows];
  const int lane = threadIdx.x & 31, warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), g = lane >> 2, c = lane & 3;
  if (lane == 0)
    for (int i = 0; i < ST; ++i) mbar_init(&bars[warp * ST + i], 1);
  fence_mbar_init();
  __syncwarp();
  pdl_wait();
  pdl_trigger();
  const int sp = (int)(blockIdx.x % p.splits), rt = (int)(blockIdx.x / p.splits % p.rtiles);
  int64_t bh = blockIdx.x / p.splits / p.rtiles, b = bh / p.c.Hkv;
  const int hk = (int)(bh - b * p.c.Hkv), Gq = p.H / p.c.Hkv, rows = p.Lq * Gq;
  const int most = p.M << p.c.log_page;
  if (p.longest_first) {  // the entry that has b longer ones before it
    int len = 0, before = 0;
    if (threadIdx.x < p.B) s_len[threadIdx.x] = len = min(max(p.lens[threadIdx.x], 0), most);
    __syncthreads();
    for (int i = 0; i < p.B; ++i) before += s_len[i] > len || (s_len[i] == len && i < threadIdx.x);
    if (threadIdx.x < p.B && before == b) s_entry = threadIdx.x;
    __syncthreads();
    b = __shfl_sync(0xffffffffu, s_entry, 0), bh = b * p.c.Hkv + hk;
  }
  const int n = p.lens ? min(max(p.lens[b], 0), most) : most;
  const int units = n / kUnit + (n % kUnit != 0);  // n + kUnit - 1 may pass 31 bits
  const int u_lo = (int)((int64_t)units * sp / p.splits), u_hi = (int)((int64_t)units * (sp + 1) / p.splits);

  // ---- copies: one elected lane asks for the codes and scales of a unit (of two pages where they have 16 tokens) ----
  unsigned char* ring = smem + warp * ST * Sh::kStage;
  uint64_t* bar = bars + warp * ST;
  const int32_t* table = p.table + b * p.M;
  const bool small = p.c.page == 16;
  const int half = lane >> 2 & 1;
  uint32_t holes = 0;  // two bits a stage: halves of a unit that are not there
  // this lane's page of unit u
  auto page_of = [&](int u) {
    return u < u_hi && u * kUnit + (small ? half * 16 : 0) < n ? table[(u * kUnit >> p.c.log_page) + (small ? half : 0)] : -1;
  };
  auto ask = [&](int s, int64_t token, auto tokens, int to) {  // from the page's token on, to the stage's
    unsigned char* dst = ring + s * Sh::kStage;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      bulk_g2s(dst + kv * Sh::kCodes + to * (D / 2), p.c.q[kv] + token * (D / 2), tokens * (D / 2), &bar[s]);
      bulk_g2s(dst + 2 * Sh::kCodes + kv * Sh::kScales + to * (D / 16),
               reinterpret_cast<const unsigned char*>(p.c.scale[kv]) + token * (D / 16), tokens * (D / 16), &bar[s]);
    }
  };
  auto fetch = [&](int u, int s, int id) {
    if (u >= u_hi) return;
    const int id0 = __shfl_sync(0xffffffffu, id, 0), id1 = small ? __shfl_sync(0xffffffffu, id, 4) : id0;
    const bool hole0 = (unsigned)id0 >= (unsigned)p.c.pages, hole1 = (unsigned)id1 >= (unsigned)p.c.pages;
    if ((hole0 || (hole1 && u * kUnit + 16 < n)) && lane == 0) record_error(p.err, HCLSM_ERR_SHAPE);
    holes = (holes & ~(3u << 2 * s)) | ((hole0 ? 1u : 0u) | (hole1 ? 2u : 0u)) << 2 * s;
    if (!tc::elect_one()) return;
    if (!small) {
      mbar_expect_tx(&bar[s], hole0 ? 0u : Sh::kStage);
      if (!hole0) ask(s, ((int64_t)id0 * p.c.Hkv + hk) * p.c.page + (u * kUnit & (p.c.page - 1)), kUnit, 0);
    } else {
      mbar_expect_tx(&bar[s], (hole0 ? 0u : Sh::kStage / 2) + (hole1 ? 0u : Sh::kStage / 2));
      if (!hole0) ask(s, ((int64_t)id0 * p.c.Hkv + hk) * 16, 16, 0);
      if (!hole1) ask(s, ((int64_t)id1 * p.c.Hkv + hk) * 16, 16, 16);
    }
  };
  const int u0 = u_lo + warp;
#pragma unroll 1
  for (int i = 0; i < ST - 1; ++i) fetch(u0 + i * kWarps, i, page_of(u0 + i * kWarps));
  int next = page_of(u0 + (ST - 1) * kWarps);

  // ---- queries: fragments of Q^T, row g of each tile, dims 8 c + i and 8 c + 4 + i of a group side by side ----
  uint32_t qb[Sh::kF32 ? 1 : RT][G][4];
  float q136[Sh::kF32 ? 1 : RT][G][2];  // -136 times the sum of a group of rows 2 c and 2 c + 1
  uint32_t* frag = reinterpret_cast<uint32_t*>(smem + (Sh::kBytes - Sh::kFrag - Sh::kWide));
  auto row_at = [&](int r) {  // a row's query, or null
    const int row = rt * kRows + r;
    return row < rows ? static_cast<const T*>(p.q.p) + b * p.q.sb + (int64_t)(row / Gq) * p.q.st +
                            (int64_t)(hk * Gq + row % Gq) * p.q.sh
                      : nullptr;
  };
  if constexpr (!Sh::kF32) {
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const T* q = row_at(g + 8 * r);
#pragma unroll
      for (int y = 0; y < G; ++y) {
        uint4 w = make_uint4(0, 0, 0, 0);
        if (q) w = *reinterpret_cast<const uint4*>(q + y * kGroup + 8 * c);
        qb[r][y][0] = __byte_perm(w.x, w.z, 0x5410), qb[r][y][1] = __byte_perm(w.x, w.z, 0x7632);
        qb[r][y][2] = __byte_perm(w.y, w.w, 0x5410), qb[r][y][3] = __byte_perm(w.y, w.w, 0x7632);
        float sum = 0.0f;
        const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) sum += __uint_as_float(v[i] << 16) + __uint_as_float(v[i] & 0xffff0000u);
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        q136[r][y][0] = -136.0f * __shfl_sync(0xffffffffu, sum, 8 * c);
        q136[r][y][1] = -136.0f * __shfl_sync(0xffffffffu, sum, 8 * c + 4);
      }
    }
  } else {
    // fragment words [piece][group][step][lane][RT][2]
    for (int i = threadIdx.x; i < G * 2 * 32; i += kThreads) {
      const int l = i & 31, step = i >> 5 & 1, y = i >> 6;
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const T* q = row_at((l >> 2) + 8 * r);
        const int d = y * kGroup + 8 * (l & 3) + 2 * step;
        uint32_t w[2][NQ];
#pragma unroll
        for (int e = 0; e < 2; ++e) pieces<NQ>(q ? (float)q[d + e] : 0.0f, q ? (float)q[d + e + 4] : 0.0f, w[e]);
#pragma unroll
        for (int k = 0; k < NQ; ++k)
          *reinterpret_cast<uint2*>(frag + ((((k * G + y) * 2 + step) * 32 + l) * RT + r) * 2) =
              make_uint2(w[0][k], w[1][k]);
      }
    }
    __syncthreads();
  }

  // ---- tokens ------------------------------------------------------------------------------
  // o[tile][r]: dims 4 g + 2 (tile % 2) (and + 1) of group tile / 2, rows 2 c and 2 c + 1 of row tile r
  float o[D / 16][RT][4] = {};
  float m[RT][2], l[RT][2];
#pragma unroll
  for (int r = 0; r < RT; ++r) m[r][0] = m[r][1] = -INFINITY, l[r][0] = l[r][1] = 0.0f;
  // Of a tile of 8 tokens, the one that is row g of K (and lane g's scores) and columns 2 c and 2 c + 1 of V^T: an order in
  // which neither keys (four rows a load's half) nor values (four tokens a load) meet in a bank with 64 dims.
  const int key = g & 1 ? (g >> 1) + 2 : (g >> 1) + 2 * (g >> 1 & 2);
  const int tok0 = c + 2 * (c & 2), tok1 = c + 2;
  float *ks = reinterpret_cast<float*>(smem + (Sh::kBytes - Sh::kWide)) + warp * 2 * kUnit * G, *vs = ks + kUnit * G;
  // a maximum stays while no score is 2^8 above it in its power: nothing overflows, and no lane asks the others each step
  const float slack = fminf(8.0f / p.c2, 3.0e38f);
  uint32_t k128 = 0x43004300u;
  asm volatile("" : "+r"(k128));
  int s = 0;
  uint32_t phase = 0;
  bool alive = true;
#pragma unroll 1
  for (int u = u0; u < u_hi; u += kWarps) {
    const int s_new = s == 0 ? ST - 1 : s - 1;
    __syncwarp();  // all lanes have left the stage that is filled now
    fetch(u + (ST - 1) * kWarps, s_new, next);
    next = page_of(u + ST * kWarps);
    if (!__all_sync(0xffffffffu, mbar_wait(&bar[s], phase))) {
      alive = false;
      break;
    }
    const unsigned char* kq = ring + s * Sh::kStage;
    const unsigned char* vq = kq + Sh::kCodes;
    if (lane < 8 * G) {  // the scales of the unit as fp32: eight a lane, keys' and then values'
      const uint4 w = *reinterpret_cast<const uint4*>(vq + Sh::kCodes + lane * 16);
      float4* to = reinterpret_cast<float4*>(ks + lane * 8);
      to[0] = make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16),
                          __uint_as_float(w.y & 0xffff0000u));
      to[1] = make_float4(__uint_as_float(w.z << 16), __uint_as_float(w.z & 0xffff0000u), __uint_as_float(w.w << 16),
                          __uint_as_float(w.w & 0xffff0000u));
    }
    __syncwarp();
    const uint32_t hole = holes >> 2 * s & 3u;
    if (++s == ST) s = 0, phase ^= 1;
    const int left = n - u * kUnit;
    uint32_t valid = left >= kUnit ? 0xffffffffu : (1u << left) - 1u;
    if (hole) valid &= small ? (hole & 1 ? 0xffff0000u : ~0u) & (hole & 2 ? 0xffffu : ~0u) : hole & 1 ? 0u : ~0u;
    if (valid == 0) continue;

    float sc[2][RT][4];  // 16 tokens: lane's tokens key and key + 8, rows 2 c and 2 c + 1
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int t = 16 * h + key;
      float f0[G], f1[G];
      scales<G>(ks + t * G, f0);
      scales<G>(ks + (t + 8) * G, f1);
      const uint32_t* row0 = reinterpret_cast<const uint32_t*>(kq + t * (D / 2));
      const uint32_t* row1 = row0 + D;
#pragma unroll
      for (int y = 0; y < G; ++y) {
        uint32_t x0, x1;  // this lane's eight codes of the group: dims 8 c + i (low half), 8 c + 4 + i
        if (y / 2 * 64 + 64 <= D) {
          const uint2 w0 = *reinterpret_cast<const uint2*>(row0 + y / 2 * 8 + 2 * c);
          const uint2 w1 = *reinterpret_cast<const uint2*>(row1 + y / 2 * 8 + 2 * c);
          x0 = __byte_perm(w0.x, w0.y, y & 1 ? 0x7632 : 0x5410);
          x1 = __byte_perm(w1.x, w1.y, y & 1 ? 0x7632 : 0x5410);
        } else {
          x0 = row0[y / 2 * 8 + c], x1 = row1[y / 2 * 8 + c];
        }
        float d[RT][4];
#pragma unroll
        for (int step = 0; step < 2; ++step) {
          const int i = 8 * step;
          if constexpr (Sh::kF32) {
            const uint32_t a[4] = {centred(x0 >> i, k128), centred(x1 >> i, k128), centred(x0 >> (i + 4), k128),
                                   centred(x1 >> (i + 4), k128)};
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
              for (int k = 0; k < NQ; ++k) {
                const uint2 w = *reinterpret_cast<const uint2*>(frag + ((((k * G + y) * 2 + step) * 32 + lane) * RT + r) * 2);
                if (step == 0 && k == 0) mma(d[r], a, w.x, w.y, 0.0f, 0.0f, 0.0f, 0.0f);
                else mma(d[r], a, w.x, w.y);
              }
          } else {
            const uint32_t a[4] = {biased(x0 >> i, k128), biased(x1 >> i, k128), biased(x0 >> (i + 4), k128),
                                   biased(x1 >> (i + 4), k128)};
#pragma unroll
            for (int r = 0; r < RT; ++r) {
              if (step == 0)
                mma(d[r], a, qb[r][y][0], qb[r][y][1], q136[r][y][0], q136[r][y][1], q136[r][y][0], q136[r][y][1]);
              else
                mma(d[r], a, qb[r][y][2], qb[r][y][3]);
            }
          }
        }
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float f = e < 2 ? f0[y] : f1[y];
            sc[h][r][e] = y == 0 ? d[r][e] * f : fmaf(d[r][e], f, sc[h][r][e]);
          }
      }
    }
    if (valid != 0xffffffffu) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!(valid >> (16 * h + key + (e < 2 ? 0 : 8)) & 1u)) sc[h][r][e] = -INFINITY;
    }
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      float top[2];
#pragma unroll
      for (int e = 0; e < 2; ++e)
        top[e] = fmaxf(fmaxf(sc[0][r][e], sc[0][r][e + 2]), fmaxf(sc[1][r][e], sc[1][r][e + 2]));
      if (__any_sync(0xffffffffu, top[0] > m[r][0] + slack || top[1] > m[r][1] + slack)) {
        float f[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int x = 4; x <= 16; x <<= 1) top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], x));
          const float was = m[r][e];
          m[r][e] = fmaxf(was, top[e]);
          f[e] = was == m[r][e] ? 1.0f : ex2((was - m[r][e]) * p.c2);
          l[r][e] *= f[e];
        }
#pragma unroll
        for (int j = 0; j < D / 16; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[j][r][e] *= f[e & 1];
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float base = m[r][e] == -INFINITY ? 0.0f : -m[r][e] * p.c2;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int k = 0; k < 4; k += 2) {
            sc[h][r][k + e] = ex2(fmaf(sc[h][r][k + e], p.c2, base));
            l[r][e] += sc[h][r][k + e];
          }
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {  // 16 tokens
      float f0[G], f1[G];
      scales<G>(vs + (16 * h + key) * G, f0);
      scales<G>(vs + (16 * h + key + 8) * G, f1);
      if (valid != 0xffffffffu) {  // what is not there may have any scale, NaN too
        const bool a = valid >> (16 * h + key) & 1u, z = valid >> (16 * h + key + 8) & 1u;
#pragma unroll
        for (int y = 0; y < G; ++y) f0[y] = a ? f0[y] : 0.0f, f1[y] = z ? f1[y] : 0.0f;
      }
      const uint32_t* w0 = reinterpret_cast<const uint32_t*>(vq + (16 * h + tok0) * (D / 2));
      const uint32_t* w1 = reinterpret_cast<const uint32_t*>(vq + (16 * h + tok1) * (D / 2));
#pragma unroll
      for (int y = 0; y < G; ++y) {
        const bool paired = y / 2 * 64 + 64 <= D;
        const int at = y / 2 * 8 + (paired ? g : g >> 1);
        const uint32_t sel = (paired ? y & 1 : g & 1) ? 0x7632 : 0x5410;
        const uint32_t x0 = __byte_perm(w0[at], w1[at], sel), x1 = __byte_perm(w0[at + D], w1[at + D], sel);
        uint32_t pb[RT][NQ][2];
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          uint32_t v[2][NQ];
          pieces<NQ>(sc[h][r][0] * f0[y], sc[h][r][1] * f0[y], v[0]);
          pieces<NQ>(sc[h][r][2] * f1[y], sc[h][r][3] * f1[y], v[1]);
#pragma unroll
          for (int k = 0; k < NQ; ++k) pb[r][k][0] = turned(v[0][k]), pb[r][k][1] = turned(v[1][k]);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t a[4] = {centred(x0 >> 8 * i, k128), centred(x0 >> (8 * i + 4), k128), centred(x1 >> 8 * i, k128),
                                 centred(x1 >> (8 * i + 4), k128)};
#pragma unroll
          for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int k = 0; k < NQ; ++k) mma(o[2 * y + i][r], a, pb[r][k][0], pb[r][k][1]);
        }
      }
    }
  }
  if (!alive) {  // a wait ran out: the copies in flight end before the block's memory does
    if (lane == 0) record_error(p.err, HCLSM_ERR_TIMEOUT);
    for (int i = 0; i < ST; ++i) mbar_wait(&bar[i], phase ^ (i < s ? 1u : 0u));
  }

  // ---- merge the warps, in order -----------------------------------------------------------
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float sum = l[r][e];
#pragma unroll
      for (int x = 4; x <= 16; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
      if (g == 0) s_m[warp][8 * r + 2 * c + e] = m[r][e], s_l[warp][8 * r + 2 * c + e] = sum;
    }
  __syncthreads();  // the rings are done with
  float* part = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int j = 0; j < D / 16; ++j)
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        part[(warp * kRows + 8 * r + 2 * c + (e & 1)) * D + j / 2 * kGroup + 4 * g + 2 * (j & 1) + (e >> 1)] = o[j][r][e];
  if (threadIdx.x < kRows) {
    const int r = threadIdx.x;
    float top = -INFINITY, sum = 0.0f;
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_m[w][r]);
    for (int w = 0; w < kWarps; ++w) {
      // a part without a maximum holds zeros, or NaN that has to stay
      const float f = s_m[w][r] == -INFINITY ? 1.0f : ex2((s_m[w][r] - top) * p.c2);
      s_w[w][r] = f;
      sum += f * s_l[w][r];
    }
    if (p.cluster) {
      s_m[0][r] = top, s_l[0][r] = sum;
    } else if (p.splits > 1) {
      p.part_ml[((bh * p.rtiles + rt) * p.splits + sp) * kRows + r] = make_float2(top, sum);
    } else {
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
      for (int w = 0; w < kWarps; ++w) s_w[w][r] *= inv;
    }
  }
  __syncthreads();
  auto row_out = [&](int row) {
    return static_cast<T*>(p.o) + ((b * p.Lq + row / Gq) * p.H + hk * Gq + row % Gq) * (int64_t)D;
  };
  for (int i = threadIdx.x; i < kRows * D; i += kThreads) {
    const int r = i / D, d = i % D, row = rt * kRows + r;
    if (row >= rows) break;
    float a = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) a += s_w[w][r] * part[(w * kRows + r) * D + d];
    if (p.cluster)
      part[i] = a;  // over warp 0's, which this thread has read
    else if (p.splits > 1)
      p.part_o[(((bh * p.rtiles + rt) * p.splits + sp) * kRows + r) * D + d] = a;
    else
      io<T>::st(row_out(row) + d, a);
  }
  if (p.cluster) {
    namespace cg = cooperative_groups;
    const cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    // the cluster's blocks share out the values; each is joined in the order of the splits
    for (int i = sp * kThreads + threadIdx.x; i < kRows * D; i += p.splits * kThreads) {
      const int r = i / D, row = rt * kRows + r;
      if (row >= rows) break;
      float top = -INFINITY, sum = 0.0f, a = 0.0f;
      for (int k = 0; k < p.splits; ++k) top = fmaxf(top, cluster.map_shared_rank(&s_m[0][0], k)[r]);
      for (int k = 0; k < p.splits; ++k) {
        const float m1 = cluster.map_shared_rank(&s_m[0][0], k)[r];
        const float f = m1 == -INFINITY ? 1.0f : ex2((m1 - top) * p.c2);
        sum += f * cluster.map_shared_rank(&s_l[0][0], k)[r];
        a += f * cluster.map_shared_rank(part, k)[i];
      }
      io<T>::st(row_out(row) + i % D, sum == 0.0f ? 0.0f : a * (1.0f / sum));
    }
    cluster.sync();  // no block leaves while others read its parts
  }
}

// One warp a row: the splits' parts, in order.
template <typename T, int D, int kRows>
__global__ void __launch_bounds__(kThreads) join_kernel(const __grid_constant__ Attn p) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  const int Gq = p.H / p.c.Hkv, rows = p.Lq * Gq;
  const int64_t at = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (at >= (int64_t)p.B * p.c.Hkv * rows) return;
  const int64_t bh = at / rows, b = bh / p.c.Hkv;
  const int row = (int)(at % rows), h = (int)(bh % p.c.Hkv) * Gq + row % Gq;
  const int64_t part = ((bh * p.rtiles + row / kRows) * p.splits) * kRows + row % kRows;
  float m = -INFINITY;
  for (int s = lane; s < p.splits; s += 32) m = fmaxf(m, p.part_ml[part + (int64_t)s * kRows].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  float l = 0.0f, acc[D / 32] = {};
#pragma unroll 4
  for (int s = 0; s < p.splits; ++s) {
    const float2 ml = p.part_ml[part + (int64_t)s * kRows];
    const float f = ml.x == -INFINITY ? 1.0f : ex2((ml.x - m) * p.c2);
    l += f * ml.y;
    const float* o = p.part_o + (part + (int64_t)s * kRows) * D;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) acc[i] += f * o[lane + 32 * i];
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  T* out = static_cast<T*>(p.o) + ((b * p.Lq + row / Gq) * p.H + h) * (int64_t)D;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) io<T>::st(out + lane + 32 * i, acc[i] * inv);
}

// Rows a block: 8 where that is all, else 16, which share the work of unpacking the codes.
int row_tile(const Attn& p) { return (int64_t)p.Lq * (p.H / p.c.Hkv) <= 8 ? 8 : 16; }

// Whole waves of resident blocks; a block's share is its own sequence's, so more waves even unequal lengths out, down
// to 1024 tokens a block (a block writes its rows in fp32 for the join).
void plan(Attn& p, int dtype) {
  const int64_t rows = (int64_t)p.Lq * (p.H / p.c.Hkv), keys = (int64_t)p.M << p.c.log_page;
  p.rtiles = (int)((rows + row_tile(p) - 1) / row_tile(p));
  const int64_t base = (int64_t)p.B * p.c.Hkv * p.rtiles;
  const int per_sm = blocks_per_sm(dtype == HCLSM_F32, p.c.D, row_tile(p) / 8);
  int64_t s = 1;
  for (int waves = 1; waves <= kWaves; ++waves) {
    const int64_t n = base > 0 ? (int64_t)num_sms() * per_sm * waves / base : 1;
    if (n > 1 && (waves == 1 || keys / n >= kMinKeys)) s = n;
  }
  const int64_t most = (keys + 127) / 128;
  if (s > most) s = most;
  // Up to eight splits join in their cluster's shared memory.  Nine to sixteen are made eight, fewer waves than above: up to
  // some 16384 tokens a second launch costs more (slots, write and attention of one token over 8 x 2048, 6 heads of 64: 16.5 us
  // with it, 12.5 without; 20 x 16384, 8 key heads of 128: 91 and 86), for longer ones less (20 x 65536: 258 and 271).
  if (s <= 16) s = s < 8 ? s : 8;
  p.splits = s < 1 ? 1 : (int)s;
  p.cluster = p.splits > 1 && p.splits <= 8;
  // Blocks of unequal lengths in several waves: the long ones first, so that the last to run are short.
  p.longest_first = p.lens && p.B > 1 && p.B <= kThreads && base * p.splits > (int64_t)num_sms() * per_sm;
}

size_t attn_workspace(const Attn& a, int dtype) {
  Attn p = a;
  plan(p, dtype);
  if (p.splits <= 1 || p.cluster) return 0;
  return (size_t)p.B * p.c.Hkv * p.rtiles * p.splits * row_tile(p) * (p.c.D * sizeof(float) + sizeof(float2));
}

template <typename T, int D, int RT>
int launch(Attn& p, void* ws, cudaStream_t st) {
  using Sh = Shape<T, D, RT>;
  const int64_t grid = (int64_t)p.B * p.c.Hkv * p.rtiles * p.splits, rows = (int64_t)p.B * p.H * p.Lq;
  if (grid > 0x7fffffff || rows / kWarps > 0x7ffffff0) return HCLSM_ERR_SHAPE;
  if (p.splits > 1 && !p.cluster) {
    p.part_ml = static_cast<float2*>(ws);
    p.part_o = reinterpret_cast<float*>(p.part_ml + grid * Sh::kRows);
  }
  auto f = attn_kernel<T, D, RT>;
  if (!set_smem_limit(reinterpret_cast<const void*>(f), Sh::kBytes)) return HCLSM_ERR_LAUNCH;
  if (p.cluster) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = (unsigned)grid, cfg.blockDim = kThreads, cfg.dynamicSmemBytes = Sh::kBytes, cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)p.splits, attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr, cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, f, p) == cudaSuccess ? HCLSM_OK : HCLSM_ERR_LAUNCH;
  }
  if (const int rc = launch_pdl(f, (unsigned)grid, kThreads, Sh::kBytes, st, p)) return rc;
  if (p.splits <= 1) return HCLSM_OK;
  return launch_pdl(join_kernel<T, D, Sh::kRows>, (unsigned)((rows + kWarps - 1) / kWarps), kThreads, 0, st, p);
}

template <typename T, int D>
int launch_rows(Attn& p, void* ws, cudaStream_t st) {
  return row_tile(p) == 8 ? launch<T, D, 1>(p, ws, st) : launch<T, D, 2>(p, ws, st);
}

int attn(Attn p, int dtype, void* ws, cudaStream_t st) {
  plan(p, dtype);
  const bool f = dtype == HCLSM_F32;
  switch (p.c.D) {
    case 32: return f ? launch_rows<float, 32>(p, ws, st) : launch_rows<__nv_bfloat16, 32>(p, ws, st);
    case 64: return f ? launch_rows<float, 64>(p, ws, st) : launch_rows<__nv_bfloat16, 64>(p, ws, st);
    case 96: return f ? launch_rows<float, 96>(p, ws, st) : launch_rows<__nv_bfloat16, 96>(p, ws, st);
    default: return f ? launch_rows<float, 128>(p, ws, st) : launch_rows<__nv_bfloat16, 128>(p, ws, st);
  }
}

}  // namespace kv4
}  // namespace hclsm
