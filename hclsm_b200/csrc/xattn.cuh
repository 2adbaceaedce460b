// What the cross-attention kernels share.
//
//   s_ij = scale q_i . k_j,   p_ij = exp(s_ij) / sum_j exp(s_ij) over the allowed keys j,   o_i = sum_j p_ij v_j
//
// A key is allowed when its index is below its batch entry's length and its
// mask byte is not zero.  A row with no allowed key gives 0 (and zero
// gradients).  Keys and values that are not allowed are never arithmetic
// operands: they are replaced by zeros on their way in, because 0 * NaN is NaN.
// Softmax runs in base 2 (scale * log2 e folded into one factor).  The forward
// keeps lse2 = max + log2(sum) for the backward, +inf for an empty row, so that
// exp2(s - lse2) is 0 there.  With delta_i = sum_d do_id o_id:
//   ds_ij = p_ij (do_i . v_j - delta_i)
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,  dv_j = sum_i p_ij do_i
// (dk and dv also over the query heads that share the key head).
#pragma once
#include "common.cuh"

namespace hclsm {
int* device_err_ptr();
int num_sms();
bool set_smem_limit(const void* fn, size_t bytes);

namespace xattn {

struct View {
  const void* p;
  int64_t sb, st, sh;  // elements
};
// A caller's (B, L, H, D) tensor; a dim of one is never stepped over, whatever its stride.
inline View view(const hclsm_view& v, int B, int L, int H) {
  return View{v.p, B > 1 ? v.sb : 0, L > 1 ? v.st : 0, H > 1 ? v.sh : 0};
}

struct Params {
  View q, k, v, dout;          // (B, L, H, D), innermost dense
  void *o, *dq, *dk, *dv;      // dense (B, L, H, D)
  float* lse2;                 // (B, H, Lq)
  __nv_bfloat16* lo;           // bf16 calls, (B, Lq, H, D) or null: o before rounding minus o
  float* delta;                // (B, H, Lq)
  float* part;                 // the mma.sync dk, dv kernel: (2, G, B, Lk, Hkv, D) of each query head, or null
  const int32_t* lens;         // (B) or null
  const uint8_t* mask;         // (B, Lk) rows mask_sb apart, or null
  int64_t mask_sb;
  int B, Lq, Lk, H, Hkv, D;
  float scale;
  int* err;
};

// Keys of batch entry b that can be allowed at all.
__device__ __forceinline__ int key_count(const Params& p, int64_t b) {
  return p.lens ? min(max(p.lens[b], 0), p.Lk) : p.Lk;
}
// What rounding to bf16 takes from v.
__device__ __forceinline__ float rounding(float v) { return v - __bfloat162float(__float2bfloat16_rn(v)); }
__device__ __forceinline__ bool key_ok(const Params& p, int64_t b, int n, int j) {
  return j < n && (!p.mask || p.mask[b * p.mask_sb + j]);
}

// bf16 on the 5th-generation tensor cores (xattn_tc.cu), where tc_ok.
bool tc_ok(const Params& p, bool bwd);
size_t tc_workspace(const Params& p);
int tc_fwd(const Params& p, void* ws, cudaStream_t st);
int tc_bwd(const Params& p, void* ws, cudaStream_t st);
// Few query rows, the keys split over blocks (attn_split.cu).
size_t split_workspace(const Params& p, int dtype);
int split_fwd(const Params& p, int dtype, void* ws, cudaStream_t st);

}  // namespace xattn
}  // namespace hclsm
