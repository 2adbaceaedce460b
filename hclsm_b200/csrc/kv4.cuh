// What the kernels of the paged 4-bit state cache share.
//
// A token's dims of one head are groups of 32 with a bf16 scale each; a value is (code - 8) * scale, code 0 to 15.
// The scale is the value of largest magnitude over -8, so that value is held as -8 (exactly, where it is a bf16
// number) and the step is a sixteenth of the symmetric range: a seventh finer than +-7 steps, for a clipped 8.
// The codes of dims d to d + 3 and d + 32 to d + 35 of 64 share a 32-bit word: the halves of one word then belong
// to different scales and the halves of two words to the same one, which is how the attention's products take them.
#pragma once
#include "xattn.cuh"

namespace hclsm {
namespace kv4 {

constexpr int kGroup = 32;

struct Cache {
  uint8_t* q[2];      // keys, values: (pages, Hkv, page, D / 2)
  uint16_t* scale[2]; // bf16 (pages, Hkv, page, D / 32)
  int pages, Hkv, page, log_page, D;
};

inline Cache cache(const hclsm_kv4_cache* c) {
  Cache r = {{c->k, c->v}, {c->k_scale, c->v_scale}, c->pages, c->Hkv, c->page, 0, c->D};
  while ((1 << r.log_page) < c->page) ++r.log_page;
  return r;
}

struct Attn {
  Cache c;
  xattn::View q;      // (B, Lq, H, D)
  void* o;            // dense
  const int32_t *table, *lens;
  int B, M, Lq, H;
  int splits, rtiles;
  int cluster;        // the splits of a row are one cluster, whose blocks join them
  int longest_first;  // entries in the order of their lengths
  float* part_o;      // (B * Hkv * rtiles, splits, 16, D)
  float2* part_ml;    // (B * Hkv * rtiles, splits, 16): max, sum
  float c2;           // scale * log2 e
  int* err;
};

size_t attn_workspace(const Attn& p, int dtype);
int attn(Attn p, int dtype, void* ws, cudaStream_t st);

}  // namespace kv4
}  // namespace hclsm
