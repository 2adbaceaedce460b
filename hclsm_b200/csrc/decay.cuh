// Linear attention whose state forgets at a rate of each head.
//
//   S_t = g S_{t-1} + k_t^T v_t,   o_t = scale q_t S_t,   g = exp(log_decay) in [0, 1],   S_{-1} the given state or 0
//
// Everything is one kind of pass over x, k, v (rows of a head's tokens) in either direction of time:
//
//   T <- g T + w k_t^T v_t,   y_t = f x_t T      t ascending or, reversed, descending from the last valid token
//
//   forward:  (x, k, v) = (q, k, v), ascending from S_{-1}, w = 1, f = scale; T ends as the new state
//   dq:       (dO, v, k), ascending from S_{-1}^T, w = 1, f = scale
//   dv:       (k, q, dO), descending from dS, w = scale, f = 1, where the first token meets T without a decay, and T
//             ends as g T = dS_{-1}
//   dk:       (v, dO, q), descending from dS^T, w = scale, f = 1
//
// (dS knows no scale: a T that is multiplied by it at the end would have to start from dS / scale, which may overflow.)
//
// By chunks of C tokens, i and j a token's place among the m valid ones in the pass's order and r = 1 where reversed:
//
//   y_i = f [ sum_{j <= i} w g^{i-j} (x_i . k_j) v_j  +  g^{i+1-r} x_i T ],   T <- g^m T + sum_j w g^{m-1-j+r} k_j^T v_j
//
// Chunks lie on multiples of C in memory in both directions, so the incomplete one is the last one.  Where the heads
// do not fill the GPU their tokens are cut into segments of whole chunks: the segments' own sums (sums pass), their
// running combination (join kernel), then the segments side by side, each from its own state.
#pragma once
#include "xattn.cuh"

namespace hclsm {
namespace decay {

using xattn::View;

struct Pass {
  View x, k, v;               // (B, L, H, Dk), (B, L, H, Dk), (B, L, H, Dv), innermost dense
  void* y;                    // dense (B, L, H, Dv)
  const float* log_decay;     // (H)
  const float* init;          // (B, H, Dk, Dv), or transposed, or null
  float* last;                // the same for the final state
  const int32_t* lens;        // (B) or null
  float* part;                // (B * H, segs, Dk, Dv): sums, then the segments' first states
  int init_t;                 // init is (B, H, Dv, Dk)
  float w, f;                 // factors of the tokens' weights and of y
  int rev;
  int B, L, H, Dk, Dv;
  int segs, seg_chunks;       // segments a head, chunks of a segment
  int* err;
};

// log2 of a head's decay, at most 0 (NaN stays).  Where it is below -200 (-inf, which would be NaN where the exponent is
// 0) one token forgets all in fp32 either way.
__device__ __forceinline__ float log2_decay(const float* log_decay, int h) {
  float l = log_decay[h] * kLog2e;
  l = l > 0.0f ? 0.0f : l;
  return l < -200.0f ? -200.0f : l;
}
// g^n.  A chunk's factor meets the state once a chunk, so its error adds up over as many chunks as the head remembers:
// in 64 bits, as two fp32 parts.
__device__ __forceinline__ float2 chunk_decay(const float* log_decay, int h, int n) {
  double l = (double)log_decay[h];
  l = l > 0.0 ? 0.0 : l;
  l = l < -1e30 ? -1e30 : l;
  const double g = exp(l * n);
  const float hi = (float)g;
  return make_float2(hi, (float)(g - (double)hi));
}
// Chunks of n tokens; n + chunk - 1 may pass 31 bits.
__host__ __device__ __forceinline__ int chunks_of(int n, int chunk) { return n / chunk + (n % chunk != 0); }
__device__ __forceinline__ int length(const Pass& p, int64_t b) {
  return p.lens ? min(max(p.lens[b], 0), p.L) : p.L;
}

// Passes over the same sizes that run side by side in one launch: a block's pass is blockIdx.x % n.
constexpr int kMost = 3;
struct Batch {
  Pass p[kMost];
  int n;
};

// Segments of a head, as their cost has it, in chunks' times of a block that is alone on its SM: with the segments' own
// sums a chunk costs `twice`, `crowd` as much where blocks share an SM; the sums' and the join's launches cost `fixed`, and
// what they move `load` a block of every SM.  Measured in bf16 (1.9, 1.4, 4, 4; us, whole against segments): 6 heads of 64,
// 8 chunks 20 against 17 in eight, 32 chunks 67 against 24 in sixteen and 31 in 32; 48 heads of 64, 16 chunks 36 against
// 40 in six, 32 chunks 69 against 58 in six; 16 heads of 128, 8 chunks 27 against 38 in eight, 16 chunks 48 against 43;
// 64 heads of 128, 128 chunks 348 against 377 in two.
inline void cut(Batch& b, int chunk, float twice, float crowd, float fixed, float load, int64_t have, int64_t room) {
  const int chunks = chunks_of(b.p[0].L, chunk), sms = num_sms();
  auto shared = [&](int64_t blocks) { return blocks > sms ? crowd : 1.0f; };
  int best = chunks > 1 ? chunks : 1;  // chunks of a segment
  float least = (float)chunks * shared(have);
  for (int64_t s = 2; s <= chunks && s * have <= room; ++s) {
    const int each = (int)((chunks + s - 1) / s);
    const float cost = fixed + load * (float)(s * have) / (float)sms + twice * (float)each * shared(s * have);
    if (cost < least) least = cost, best = each;
  }
  for (int i = 0; i < b.n; ++i) b.p[i].seg_chunks = best, b.p[i].segs = chunks > 0 ? (chunks + best - 1) / best : 1;
}
// Bytes of all passes' parts, and where each one's are.
inline size_t parts(Batch& b, void* ws) {
  size_t at = 0;
  for (int i = 0; i < b.n; ++i) {
    Pass& p = b.p[i];
    p.part = reinterpret_cast<float*>(static_cast<char*>(ws) + at);
    if (p.segs > 1) at += ((size_t)p.B * p.H * p.segs * p.Dk * p.Dv * sizeof(float) + 15) & ~(size_t)15;
  }
  return at;
}

int join(const Batch& b, int chunk, cudaStream_t st);

// bf16 on the 5th-generation tensor cores (decay_tc.cu), where tc_ok.
bool tc_ok(const Batch& b);
void tc_cut(Batch& b);
int tc_run(const Batch& b, cudaStream_t st);

}  // namespace decay
}  // namespace hclsm
