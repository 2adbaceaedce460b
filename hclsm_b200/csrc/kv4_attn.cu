// Attention of few query rows over the paged 4-bit state cache.
//
// The rows that share a key head (tokens x query heads of the group) form the M = 16 side of mma.sync m16n8k16
// products; a warp takes 32 tokens a step and keeps its own running maximum, sum and output.  Each warp has a
// ring of stages of its own, filled by bulk copies that its first lane asks for (a page of one head is contiguous):
// no barrier between warps until the merge.
//
// A contraction's index can run in any order, so the products take the codes as they lie: two words' halves of the same
// 32 dims (or of two tokens) side by side, four bits at a time, 0x4300 | code = 128 + code in bf16.
//   S = Q K^T by groups of 32 dims, each times its key's scale: the 136 = 128 + 8 in every operand is taken off by
//   starting the sum at -136 times the row's sum of q in the group (fp32 states: off every operand instead,
//   their scores would lose 5 bits).
//   O += P V, P times the value's scale of the group before it is rounded to bf16: the codes are exact, so a weight
//   is rounded once.  The 136 comes off the operand (summed over a history it would drown the values).
// fp32 states: queries and weights as three bf16 pieces, whose products with exact codes are summed in fp32.
#include "kv4.cuh"

namespace hclsm {
namespace kv4 {

constexpr int kWarps = 4, kThreads = kWarps * 32, kRows = 16, kUnit = 32;
constexpr int kWaves = 4, kMinKeys = 1024;

template <typename T, int D> struct Shape {
  static constexpr bool kF32 = sizeof(T) == 4;
  static constexpr int kNQ = kF32 ? 3 : 1;  // bf16 pieces of a query or weight
  static constexpr int kG = D / kGroup;
  static constexpr int kCodes = kUnit * D / 2, kScales = kUnit * D / 16;  // bytes
  static constexpr int kStage = 2 * (kCodes + kScales);
  static constexpr int kStages = 4;
  static constexpr int kFrag = kF32 ? kNQ * kG * 2 * 32 * 16 : 0;  // query fragments of fp32 states
  static constexpr int kMerge = kWarps * kRows * D * 4;
  static constexpr int kRing = kWarps * kStages * kStage;
  static constexpr int kBytes = (kRing > kMerge ? kRing : kMerge) + kFrag;
  static constexpr int kPerSm = kF32 ? 2 : D <= 64 ? 4 : 3;
};

__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
      "%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
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
// Bits 0-3 and 16-19 as packed bf16: 128 + code, and code - 8.
__device__ __forceinline__ uint32_t biased(uint32_t x) { return (x & 0x000f000fu) | 0x43004300u; }
__device__ __forceinline__ uint32_t centred(uint32_t x) {
  const uint32_t b = biased(x), k = 0x43084308u;
  const __nv_bfloat162 r =
      __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&b), *reinterpret_cast<const __nv_bfloat162*>(&k));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// A token's scales of all groups.
template <int G> __device__ __forceinline__ void scales(const unsigned char* at, float (&s)[G]) {
  if constexpr (G == 4) {
    const uint2 w = *reinterpret_cast<const uint2*>(at);
    s[0] = __uint_as_float(w.x << 16), s[1] = __uint_as_float(w.x & 0xffff0000u);
    s[2] = __uint_as_float(w.y << 16), s[3] = __uint_as_float(w.y & 0xffff0000u);
  } else if constexpr (G == 2) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(at);
    s[0] = __uint_as_float(w << 16), s[1] = __uint_as_float(w & 0xffff0000u);
  } else {
#pragma unroll
    for (int i = 0; i < G; ++i)
      s[i] = __uint_as_float((uint32_t)reinterpret_cast<const uint16_t*>(at)[i] << 16);
  }
}

// NR 1: at most 8 rows, the upper half of the products' rows is empty.
template <typename T, int D, int NR>
__global__ void __launch_bounds__(kThreads, Shape<T, D>::kPerSm) attn_kernel(const __grid_constant__ Attn p) {
  using Sh = Shape<T, D>;
  constexpr int G = Sh::kG, NQ = Sh::kNQ, ST = Sh::kStages;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ uint64_t bars[kWarps * ST];
  __shared__ float s_m[kWarps][kRows], s_l[kWarps][kRows], s_w[kWarps][kRows];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  if (lane == 0)
    for (int i = 0; i < ST; ++i) mbar_init(&bars[warp * ST + i], 1);
  fence_mbar_init();
  __syncwarp();
  pdl_wait();
  pdl_trigger();
  const int sp = (int)(blockIdx.x % p.splits), rt = (int)(blockIdx.x / p.splits % p.rtiles);
  const int64_t bh = blockIdx.x / p.splits / p.rtiles, b = bh / p.c.Hkv;
  const int hk = (int)(bh - b * p.c.Hkv), Gq = p.H / p.c.Hkv, rows = p.Lq * Gq;
  const int n = p.lens ? min(max(p.lens[b], 0), p.M << p.c.log_page) : p.M << p.c.log_page;
  const int units = (n + kUnit - 1) / kUnit;
  const int u_lo = (int)((int64_t)units * sp / p.splits), u_hi = (int)((int64_t)units * (sp + 1) / p.splits);

  // ---- copies ------------------------------------------------------------------------------
  unsigned char* ring = smem + warp * ST * Sh::kStage;
  uint64_t* bar = bars + warp * ST;
  const int32_t* table = p.table + b * p.M;
  const bool small = p.c.page == 16;  // a unit is two pages
  uint32_t holes = 0;                 // two bits a stage: halves of a unit that are not there
  // the page numbers of unit u (loaded by all lanes alike)
  auto pages_of = [&](int u) {
    int2 r = make_int2(-1, -1);
    if (u < u_hi) {
      const int at = u * kUnit >> p.c.log_page;
      r.x = table[at];
      if (small && u * kUnit + 16 < n) r.y = table[at + 1];
    }
    return r;
  };
  auto fetch = [&](int u, int s, int2 id) {
    if (u >= u_hi) return;
    const bool a = (unsigned)id.x < (unsigned)p.c.pages, z = small && (unsigned)id.y < (unsigned)p.c.pages;
    if (lane == 0 && (!a || (small && !z && u * kUnit + 16 < n))) record_error(p.err, HCLSM_ERR_SHAPE);
    const uint32_t hole = a ? (small && !z ? 2u : 0u) : (z ? 1u : 3u);
    holes = (holes & ~(3u << 2 * s)) | hole << 2 * s;
    if (lane != 0) return;
    const int half = small ? 2 : 1, tokens = kUnit / half;
    unsigned char* to = ring + s * Sh::kStage;
    mbar_expect_tx(&bar[s], (uint32_t)((a ? 1 : 0) + (z ? 1 : 0)) * (Sh::kStage / half));
    for (int i = 0; i < half; ++i) {
      if (!(i ? z : a)) continue;
      const int64_t at = ((int64_t)(i ? id.y : id.x) * p.c.Hkv + hk) * p.c.page + (small ? 0 : u * kUnit & (p.c.page - 1));
      const int codes = tokens * D / 2, sc = tokens * D / 16;
      bulk_g2s(to + i * codes, p.c.q[0] + at * (D / 2), codes, &bar[s]);
      bulk_g2s(to + Sh::kCodes + i * codes, p.c.q[1] + at * (D / 2), codes, &bar[s]);
      bulk_g2s(to + 2 * Sh::kCodes + i * sc, p.c.scale[0] + at * (D / kGroup), sc, &bar[s]);
      bulk_g2s(to + 2 * Sh::kCodes + Sh::kScales + i * sc, p.c.scale[1] + at * (D / kGroup), sc, &bar[s]);
    }
  };
  const int u0 = u_lo + warp;
#pragma unroll
  for (int i = 0; i < ST - 1; ++i) fetch(u0 + i * kWarps, i, pages_of(u0 + i * kWarps));
  int2 next = pages_of(u0 + (ST - 1) * kWarps);

  // ---- queries -----------------------------------------------------------------------------
  uint32_t qa[Sh::kF32 ? 1 : G][2][4];
  float q136[Sh::kF32 ? 1 : G][NR];  // -136 times the row's sum of a group
  uint32_t* frag = reinterpret_cast<uint32_t*>(smem + (Sh::kBytes - Sh::kFrag));
  auto row_at = [&](int r) {  // a row's query, or null
    const int row = rt * kRows + r;
    return row < rows ? static_cast<const T*>(p.q.p) + b * p.q.sb + (int64_t)(row / Gq) * p.q.st +
                            (int64_t)(hk * Gq + row % Gq) * p.q.sh
                      : nullptr;
  };
  if constexpr (!Sh::kF32) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const T* q = r < NR ? row_at(g + 8 * r) : nullptr;
#pragma unroll
      for (int y = 0; y < G; ++y) {
        uint4 w = make_uint4(0, 0, 0, 0);
        if (q) w = *reinterpret_cast<const uint4*>(q + y * kGroup + 8 * c);
        qa[y][0][r] = __byte_perm(w.x, w.z, 0x5410), qa[y][0][2 + r] = __byte_perm(w.x, w.z, 0x7632);
        qa[y][1][r] = __byte_perm(w.y, w.w, 0x5410), qa[y][1][2 + r] = __byte_perm(w.y, w.w, 0x7632);
        if (r < NR) {
          float sum = 0.0f;
          const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) sum += __uint_as_float(v[i] << 16) + __uint_as_float(v[i] & 0xffff0000u);
          sum += __shfl_xor_sync(0xffffffffu, sum, 1);
          sum += __shfl_xor_sync(0xffffffffu, sum, 2);
          q136[y][r] = -136.0f * sum;
        }
      }
    }
  } else {
    // fragment words [piece][group][step][lane][4]
    for (int i = threadIdx.x; i < G * 2 * 32; i += kThreads) {
      const int l = i & 31, step = i >> 5 & 1, y = i >> 6;
      uint32_t w[4][NQ];
#pragma unroll
      for (int e = 0; e < 4; ++e) {  // rows l / 4 and + 8, dims 8 (l % 4) + k and + k + 4, k = 2 step + e / 2
        const T* q = row_at((l >> 2) + 8 * (e & 1));
        const int d = y * kGroup + 8 * (l & 3) + 2 * step + (e >> 1);
        pieces<NQ>(q ? (float)q[d] : 0.0f, q ? (float)q[d + 4] : 0.0f, w[e]);
      }
#pragma unroll
      for (int k = 0; k < NQ; ++k)
        *reinterpret_cast<uint4*>(frag + (((k * G + y) * 2 + step) * 32 + l) * 4) =
            make_uint4(w[0][k], w[1][k], w[2][k], w[3][k]);
    }
    __syncthreads();
  }

  // ---- tokens ------------------------------------------------------------------------------
  float o[D / 8][4] = {};
  float m[NR], l[NR];
#pragma unroll
  for (int r = 0; r < NR; ++r) m[r] = -INFINITY, l[r] = 0.0f;
  // A lane's key of a tile of 8 and its two columns' tokens: an order in which neither keys (four rows a load's half)
  // nor values (four tokens a load) meet in a bank with 64 dims.
  const int key = g & 1 ? (g >> 1) + 2 : (g >> 1) + 2 * (g >> 1 & 2);
  const int tok0 = c + 2 * (c & 2), tok1 = c + 2;
  int s = 0;
  uint32_t phase = 0;
  bool alive = true;
  for (int u = u0; u < u_hi; u += kWarps) {
    const int s_new = s == 0 ? ST - 1 : s - 1;
    __syncwarp();  // all lanes have left the stage that is filled now
    fetch(u + (ST - 1) * kWarps, s_new, next);
    next = pages_of(u + ST * kWarps);
    if (!__all_sync(0xffffffffu, mbar_wait(&bar[s], phase))) {
      alive = false;
      break;
    }
    const unsigned char* kq = ring + s * Sh::kStage;
    const unsigned char *vq = kq + Sh::kCodes, *ks = vq + Sh::kCodes, *vs = ks + Sh::kScales;
    const uint32_t hole = holes >> 2 * s & 3u;
    if (++s == ST) s = 0, phase ^= 1;
    const int left = n - u * kUnit;
    uint32_t valid = left >= kUnit ? 0xffffffffu : (1u << left) - 1u;
    if (hole) valid &= small ? (hole & 1 ? 0xffff0000u : ~0u) & (hole & 2 ? 0xffffu : ~0u) : 0u;
    if (valid == 0) continue;

    float sc[4][2 * NR];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const uint32_t* row = reinterpret_cast<const uint32_t*>(kq + (t * 8 + key) * (D / 2));
      float f0[G], f1[G];
      scales<G>(ks + (t * 8 + tok0) * (D / 16), f0);
      scales<G>(ks + (t * 8 + tok1) * (D / 16), f1);
#pragma unroll
      for (int e = 0; e < 2 * NR; ++e) sc[t][e] = 0.0f;
#pragma unroll
      for (int y = 0; y < G; ++y) {
        uint32_t x;  // this lane's eight codes of the group: dims 8 c + i (low half), 8 c + 4 + i
        if (y / 2 * 64 + 64 <= D) {
          const uint2 w = *reinterpret_cast<const uint2*>(row + y / 2 * 8 + 2 * c);
          x = __byte_perm(w.x, w.y, y & 1 ? 0x7632 : 0x5410);
        } else {
          x = row[y / 2 * 8 + c];
        }
        float d[4] = {};
        if constexpr (Sh::kF32) {
#pragma unroll
          for (int step = 0; step < 2; ++step)
#pragma unroll
            for (int k = 0; k < NQ; ++k) {
              const uint4 w = *reinterpret_cast<const uint4*>(frag + (((k * G + y) * 2 + step) * 32 + lane) * 4);
              const uint32_t a[4] = {w.x, w.y, w.z, w.w};
              mma(d, a, centred(x >> 8 * step), centred(x >> (8 * step + 4)));
            }
        } else {
#pragma unroll
          for (int e = 0; e < 2 * NR; ++e) d[e] = q136[y][e >> 1];
          mma(d, qa[y][0], biased(x), biased(x >> 4));
          mma(d, qa[y][1], biased(x >> 8), biased(x >> 12));
        }
#pragma unroll
        for (int e = 0; e < 2 * NR; ++e) sc[t][e] = fmaf(d[e], e & 1 ? f1[y] : f0[y], sc[t][e]);
      }
    }
    if (valid != 0xffffffffu) {
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int e = 0; e < 2 * NR; ++e)
          if (!(valid >> (t * 8 + (e & 1 ? tok1 : tok0)) & 1u)) sc[t][e] = -INFINITY;
    }
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      float top = fmaxf(fmaxf(sc[0][2 * r], sc[0][2 * r + 1]), fmaxf(sc[1][2 * r], sc[1][2 * r + 1]));
      top = fmaxf(top, fmaxf(fmaxf(sc[2][2 * r], sc[2][2 * r + 1]), fmaxf(sc[3][2 * r], sc[3][2 * r + 1])));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      if (__any_sync(0xffffffffu, top > m[r])) {
        const float was = m[r];
        m[r] = fmaxf(was, top);
        const float f = was == m[r] ? 1.0f : ex2((was - m[r]) * p.c2);
        l[r] *= f;
#pragma unroll
        for (int j = 0; j < D / 8; ++j) o[j][2 * r] *= f, o[j][2 * r + 1] *= f;
      }
      const float base = m[r] == -INFINITY ? 0.0f : -m[r] * p.c2;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          sc[t][2 * r + e] = ex2(fmaf(sc[t][2 * r + e], p.c2, base));
          l[r] += sc[t][2 * r + e];
        }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {  // 16 tokens
      float f[4][G];
      const int t0 = 16 * h + tok0, t1 = 16 * h + tok1;
      scales<G>(vs + t0 * (D / 16), f[0]), scales<G>(vs + t1 * (D / 16), f[1]);
      scales<G>(vs + (t0 + 8) * (D / 16), f[2]), scales<G>(vs + (t1 + 8) * (D / 16), f[3]);
      if (valid != 0xffffffffu) {  // what is not there may have any scale, NaN too
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (!(valid >> ((i & 1 ? t1 : t0) + (i & 2 ? 8 : 0)) & 1u)) {
#pragma unroll
            for (int y = 0; y < G; ++y) f[i][y] = 0.0f;
          }
      }
      const uint32_t* w0 = reinterpret_cast<const uint32_t*>(vq + t0 * (D / 2));
      const uint32_t* w1 = reinterpret_cast<const uint32_t*>(vq + t1 * (D / 2));
#pragma unroll
      for (int y = 0; y < G; ++y) {
        const bool paired = y / 2 * 64 + 64 <= D;
        const int at = y / 2 * 8 + (paired ? g : g >> 1);
        const uint32_t sel = (paired ? y & 1 : g & 1) ? 0x7632 : 0x5410;
        const uint32_t x0 = __byte_perm(w0[at], w1[at], sel), x1 = __byte_perm(w0[at + D], w1[at + D], sel);
        uint32_t a[NQ][4];
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            uint32_t v[NQ] = {};
            if (r < NR)
              pieces<NQ>(sc[2 * h + t][2 * (r < NR ? r : 0)] * f[2 * t][y],
                         sc[2 * h + t][2 * (r < NR ? r : 0) + 1] * f[2 * t + 1][y], v);
#pragma unroll
            for (int k = 0; k < NQ; ++k) a[k][2 * t + r] = v[k];
          }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t b0 = centred(x0 >> 4 * i), b1 = centred(x1 >> 4 * i);
#pragma unroll
          for (int k = 0; k < NQ; ++k) mma(o[y * 4 + i], a[k], b0, b1);
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
  for (int r = 0; r < 2; ++r) {
    float sum = r < NR ? l[r < NR ? r : 0] : 0.0f;
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    if (c == 0) s_m[warp][g + 8 * r] = r < NR ? m[r < NR ? r : 0] : -INFINITY, s_l[warp][g + 8 * r] = sum;
  }
  __syncthreads();  // the rings are done with
  float* part = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int j = 0; j < D / 8; ++j)  // tile j's columns 2 c and 2 c + 1: dims 8 c + j % 4 and + 4 of group j / 4
#pragma unroll
    for (int e = 0; e < 4; ++e)
      part[(warp * kRows + g + 8 * (e >> 1)) * D + j / 4 * kGroup + 8 * c + 4 * (e & 1) + j % 4] = o[j][e];
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
    if (p.splits > 1) {
      p.part_ml[((bh * p.rtiles + rt) * p.splits + sp) * kRows + r] = make_float2(top, sum);
    } else {
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
      for (int w = 0; w < kWarps; ++w) s_w[w][r] *= inv;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < kRows * D; i += kThreads) {
    const int r = i / D, d = i % D, row = rt * kRows + r;
    if (row >= rows) break;
    float a = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) a += s_w[w][r] * part[(w * kRows + r) * D + d];
    if (p.splits > 1)
      p.part_o[(((bh * p.rtiles + rt) * p.splits + sp) * kRows + r) * D + d] = a;
    else
      io<T>::st(static_cast<T*>(p.o) + ((b * p.Lq + row / Gq) * p.H + hk * Gq + row % Gq) * (int64_t)D + d, a);
  }
}

// One warp a row: the splits' parts, in order.
template <typename T, int D>
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

// Whole waves of resident blocks; a block's share is its own sequence's, so more waves even unequal lengths out, down
// to 1024 tokens a block (a block writes up to 16 rows of fp32 for the join).
void plan(Attn& p, int dtype) {
  const int64_t rows = (int64_t)p.Lq * (p.H / p.c.Hkv), keys = (int64_t)p.M << p.c.log_page;
  p.rtiles = (int)((rows + kRows - 1) / kRows);
  const int64_t base = (int64_t)p.B * p.c.Hkv * p.rtiles;
  const int per_sm = dtype == HCLSM_F32 ? 2 : p.c.D <= 64 ? 4 : 3;
  int64_t s = 1;
  for (int waves = 1; waves <= kWaves; ++waves) {
    const int64_t n = base > 0 ? (int64_t)num_sms() * per_sm * waves / base : 1;
    if (n > 1 && (waves == 1 || keys / n >= kMinKeys)) s = n;
  }
  const int64_t most = (keys + 127) / 128;
  if (s > most) s = most;
  p.splits = s < 1 ? 1 : (int)s;
}

size_t attn_workspace(const Attn& a, int dtype) {
  Attn p = a;
  plan(p, dtype);
  if (p.splits <= 1) return 0;
  return (size_t)p.B * p.c.Hkv * p.rtiles * p.splits * kRows * (p.c.D * sizeof(float) + sizeof(float2));
}

template <typename T, int D>
int launch(Attn& p, void* ws, cudaStream_t st) {
  using Sh = Shape<T, D>;
  const int64_t grid = (int64_t)p.B * p.c.Hkv * p.rtiles * p.splits, rows = (int64_t)p.B * p.H * p.Lq;
  if (grid > 0x7fffffff || rows / kWarps > 0x7ffffff0) return HCLSM_ERR_SHAPE;
  if (p.splits > 1) {
    p.part_ml = static_cast<float2*>(ws);
    p.part_o = reinterpret_cast<float*>(p.part_ml + grid * kRows);
  }
  auto f = (int64_t)p.Lq * (p.H / p.c.Hkv) <= 8 ? attn_kernel<T, D, 1> : attn_kernel<T, D, 2>;
  if (!set_smem_limit(reinterpret_cast<const void*>(f), Sh::kBytes)) return HCLSM_ERR_LAUNCH;
  if (const int rc = launch_pdl(f, (unsigned)grid, kThreads, Sh::kBytes, st, p)) return rc;
  if (p.splits <= 1) return HCLSM_OK;
  return launch_pdl(join_kernel<T, D>, (unsigned)((rows + kWarps - 1) / kWarps), kThreads, 0, st, p);
}

int attn(Attn p, int dtype, void* ws, cudaStream_t st) {
  plan(p, dtype);
  const bool f = dtype == HCLSM_F32;
  switch (p.c.D) {
    case 32: return f ? launch<float, 32>(p, ws, st) : launch<__nv_bfloat16, 32>(p, ws, st);
    case 64: return f ? launch<float, 64>(p, ws, st) : launch<__nv_bfloat16, 64>(p, ws, st);
    case 96: return f ? launch<float, 96>(p, ws, st) : launch<__nv_bfloat16, 96>(p, ws, st);
    default: return f ? launch<float, 128>(p, ws, st) : launch<__nv_bfloat16, 128>(p, ws, st);
  }
}

}  // namespace kv4
}  // namespace hclsm
