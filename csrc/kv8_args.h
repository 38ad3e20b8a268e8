// What the kernels of the 8-bit KV cache (kv8.cuh) are called with: plain structures and the
// launchers that csrc/kv8_ops.cpp calls once it has checked a call's tensors. No torch headers
// here or in the kernels' own files, which keeps those quick to build.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace hx {

constexpr int kKV8Block = 32;                       // tokens of a block
constexpr int kKV8Panel = kKV8Block * 64;           // values of a panel

struct KV8 {  // layouts: kv8.cuh
  uint8_t* kc;
  uint8_t* vc;
  float* ks;
  float* vs;
  __nv_bfloat16* kt;
  __nv_bfloat16* vt;
  int S, Hkv, nb, D;
  int fp8;  // codes: 0 int8, 1 e4m3

  __host__ __device__ long long head(int slot, int h) const { return (long long)slot * Hkv + h; }
  __host__ __device__ long long block(int slot, int h, int b) const { return head(slot, h) * nb + b; }
};

struct KV8AppendArgs {
  KV8 c;
  const __nv_bfloat16* k;   // row t of head h at k + t * k_row + h * k_head
  const __nv_bfloat16* v;
  long long k_row, k_head, v_row, v_head;
  int vec;                  // rows of k and v are 16-byte aligned
  int slot, p0, T, b0;      // b0: first block touched
};
cudaError_t kv8_append_launch(const KV8AppendArgs& a, cudaStream_t st);

struct KV8ReadArgs {
  KV8 c;
  __nv_bfloat16* k;         // row i of head h at k + i * k_row + h * k_head
  __nv_bfloat16* v;
  long long k_row, k_head, v_row, v_head;
  int slot, L, start, n;
};
cudaError_t kv8_read_launch(const KV8ReadArgs& a, cudaStream_t st);

struct AttnDecodeKV8Args {
  KV8 c;
  const __nv_bfloat16* proj;  // [B, ldp]: q-part (Hq*D or Hq*2D gated) | k (Hkv*D) | v (Hkv*D)
  long long ldp;
  const float* q_norm_w;      // [D] or nullptr
  const float* k_norm_w;
  const float* inv_freq;      // [rot / 2]
  const int* slots;           // [B]
  const int* pos;             // [S]
  const int* rope_delta;      // [S] rotary position - cache index, or nullptr
  int* ws;                    // word 0: errors; kKV8Err + pair: blocks done; kKV8PartAt: partials
  __nv_bfloat16* out;         // [B, Hq * D]
  int B, Hq, rot, gated;
  int G, NT, HG, per;         // G query heads of a kv head: HG groups of per (at most 8 NT)
  int vec;                    // rows of proj are 16-byte aligned
  float eps, sl2;             // scale * log2(e)
};

constexpr int kKV8Err = 64;         // words before the counters
constexpr int kKV8MaxPairs = 16384; // (sequence, kv head, head group)s of a decode call
constexpr int kKV8PartAt = kKV8Err + kKV8MaxPairs;  // the same for every batch that shares a scratch
constexpr int kKV8MaxBatch = 256;   // sequences of a decode call
constexpr int kKV8MaxCtas = 320;    // most CTAs of a decode launch, and so most partials of a pair

// Query heads of one kv head are taken in groups of 8 or 16 (the tensor cores' columns); at
// head dim 256 sixteen heads' sums do not fit a warp's registers.
inline int kv8_tiles(int G, int D) { return G > 8 && D <= 128 ? 2 : 1; }
inline int kv8_groups(int G, int D) { return (G + 8 * kv8_tiles(G, D) - 1) / (8 * kv8_tiles(G, D)); }
cudaError_t attn_decode_kv8_launch(const AttnDecodeKV8Args& a, cudaStream_t st);

struct AttnPrefillKV8Args {
  KV8 c;
  const __nv_bfloat16* q;
  const __nv_bfloat16* gate;  // row t of head h at gate + t * ldg_t + h * ldg_h, or nullptr
  __nv_bfloat16* o;
  long long ldq, ldo, ldg_t, ldg_h;
  int slot, T, p0, Hq;
  int vec_q, vec_o, vec_g;    // rows of q, o, gate are 16-byte aligned
  int NT, splits;             // row tiles of a CTA; CTAs that share a row's keys
  float* part;                // [splits, Hkv, T * G, D] where splits > 1
  float* part_ml;             // [splits, Hkv, T * G, 2]
  int* err;
  float sl2;
};
cudaError_t attn_prefill_kv8_launch(const AttnPrefillKV8Args& a, cudaStream_t st);

}  // namespace hx
