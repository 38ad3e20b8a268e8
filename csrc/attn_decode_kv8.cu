// Single-token GQA attention over the 8-bit KV cache (kv8.cuh), with the work around it in the
// same launch: q / k RMSNorm per head, rotate-half RoPE, the append of the new token (and the
// quantisation of the block that it completes), softmax attention over [0, pos] and the
// sigmoid output gate. Arguments as attn_decode.
//
// q and k stay in f32 between the norm, the rotation and the products; K is rounded to bf16
// once, as it enters the cache.
#include "attn_kv8.cuh"

namespace hx {

// RMSNorm and RoPE of one head row in shared memory (one warp).
template <int D>
HX_DEVICE void norm_rope_row(float* x, const float* w, const float* inv_freq, int rot, int p, float eps) {
  const int lane = threadIdx.x & 31;
  if (w) {
    float ss = 0.f;
    for (int d = lane; d < D; d += 32) ss += x[d] * x[d];
    const float inv = rsqrtf(warp_sum(ss) / D + eps);
    for (int d = lane; d < D; d += 32) x[d] = x[d] * inv * w[d];
    __syncwarp();
  }
  const int half = rot / 2;
  for (int i = lane; i < half; i += 32) {
    float sn, cs;
    sincosf((float)p * inv_freq[i], &sn, &cs);
    const float lo = x[i], hi = x[i + half];
    x[i] = lo * cs - hi * sn;
    x[i + half] = hi * cs + lo * sn;
  }
  __syncwarp();
}

template <int D, bool FP8>
__global__ void __launch_bounds__(128) attn_decode_kv8_kernel(AttnDecodeKV8Args a) {
  extern __shared__ __align__(16) unsigned char raw[];
  auto* s = reinterpret_cast<KV8RowsSmem<D>*>(raw);
  __shared__ float red[4];
  constexpr int NP = D / 64, ND = (D + 127) / 128;
  pdl_wait_prior();
  pdl_launch_dependents();
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, warp = tid >> 5;
  const int G = a.Hq / a.c.Hkv, qw = a.gated ? 2 * D : D;
  const __nv_bfloat16* pr = a.proj + b * a.ldp;
  const int slot = a.slots[b];
  const int p = slot >= 0 && slot < a.c.S ? a.pos[slot] : -1;
  if (p < 0 || p >= a.c.nb * kKV8Block) {  // refused: no cache access, a zero row, the error word
    for (int i = tid; i < G * D; i += 128) a.out[((long long)b * a.Hq + h * G) * D + i] = __float2bfloat16(0.f);
    if (tid == 0) atomicCAS(a.ws, 0, 6001);
    return;
  }
  const int prot = p + (a.rope_delta ? a.rope_delta[slot] : 0);
  const int L = p + 1, row = p % kKV8Block, blk = p / kKV8Block;
  // the new token enters the tail
  const __nv_bfloat16* kn = pr + a.Hq * qw + h * D;
  const __nv_bfloat16* vn = kn + a.c.Hkv * D;
  __nv_bfloat16* kt = a.c.kt + a.c.head(slot, h) * (NP * kKV8Panel);
  __nv_bfloat16* vt = a.c.vt + a.c.head(slot, h) * (NP * kKV8Panel);
  if (warp == 0) {
    for (int d = tid; d < D; d += 32) s->q[0][d] = __bfloat162float(kn[d]);
    __syncwarp();
    norm_rope_row<D>(s->q[0], a.k_norm_w, a.inv_freq, a.rot, prot, a.eps);
  }
  __syncthreads();
  for (int d = tid; d < D; d += 128) {
    kt[((d >> 6) * kKV8Block + row) * 64 + (d & 63)] = __float2bfloat16(s->q[0][d]);
    vt[d * kKV8Block + row] = vn[d];
  }
  __syncthreads();
  if (row == kKV8Block - 1) {  // complete: its codes
    for (int z = 0; z < 2; ++z) {
      const __nv_bfloat16* t = z ? vt : kt;
      float m = 0.f;
      for (int i = tid; i < D * kKV8Block; i += 128) m = fmaxf(m, kv8_mag(__bfloat162float(t[i])));
      m = warp_max(m);
      if ((tid & 31) == 0) red[warp] = m;
      __syncthreads();
      m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
      __syncthreads();
      const float inv = kv8_inv<FP8>(m);
      const long long at = a.c.block(slot, h, blk);
      uint8_t* dst = (z ? a.c.vc : a.c.kc) + at * (NP * kKV8Panel);
      for (int i = tid; i < D * kKV8Block; i += 128) dst[i] = kv8_code<FP8>(__bfloat162float(t[i]), inv);
      if (tid == 0) (z ? a.c.vs : a.c.ks)[at] = kv8_scale<FP8>(m);
    }
    __syncthreads();
  }
  for (int g0 = 0; g0 < G; g0 += kKV8Rows) {
    const int n = min(kKV8Rows, G - g0);
    __syncthreads();
    for (int g = warp; g < n; g += 4) {
      const __nv_bfloat16* q = pr + (long long)(h * G + g0 + g) * qw;
      for (int d = tid & 31; d < D; d += 32) s->q[g][d] = __bfloat162float(q[d]);
      __syncwarp();
      norm_rope_row<D>(s->q[g], a.q_norm_w, a.inv_freq, a.rot, prot, a.eps);
      for (int d = tid & 31; d < D; d += 32) s->q[g][d] *= a.sl2;
    }
    float acc[kKV8Rows][ND];
    attend_rows<D, FP8>(a.c, slot, h, L, n, [&](int) { return L; }, s, acc);
#pragma unroll
    for (int g = 0; g < kKV8Rows; ++g)
#pragma unroll
      for (int i = 0; i < ND; ++i) {
        const int d = tid + 128 * i, hq = h * G + g0 + g;
        if (g >= n || d >= D) continue;
        float o = acc[g][i];
        if (a.gated) o = o / (1.f + __expf(-__bfloat162float(pr[(long long)hq * qw + D + d])));
        a.out[((long long)b * a.Hq + hq) * D + d] = __float2bfloat16(o);
      }
  }
}

cudaError_t attn_decode_kv8_launch(const AttnDecodeKV8Args& a, cudaStream_t st) {
  cudaError_t e = cudaSuccess;
  kv8_dispatch(a.c.D, a.c.fp8, [&](auto d, auto fp8) {
    constexpr int DD = decltype(d)::value;
    auto k = attn_decode_kv8_kernel<DD, decltype(fp8)::value>;
    const size_t smem = sizeof(KV8RowsSmem<DD>);
    e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e == cudaSuccess) e = hx_launch_pdl(k, dim3((unsigned)a.c.Hkv, (unsigned)a.B), dim3(128), smem, st, a);
  });
  return e;
}

}  // namespace hx
