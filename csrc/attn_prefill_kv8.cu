// Causal GQA attention of a prompt's tokens over the 8-bit KV cache (kv8.cuh).
//
// o[t, h, :] = softmax_j(q[t, h] . k[j, h / G] * scale, j <= p0 + t) v[j, h / G]  [* sigmoid(gate)]
// for T tokens at positions p0 .. p0+T-1 whose keys and values are already in the cache.
#include "attn_kv8.cuh"

namespace hx {

template <int D, bool FP8>
__global__ void __launch_bounds__(128) attn_prefill_kv8_kernel(AttnPrefillKV8Args a) {
  extern __shared__ __align__(16) unsigned char raw[];
  auto* s = reinterpret_cast<KV8RowsSmem<D>*>(raw);
  constexpr int ND = (D + 127) / 128;
  pdl_wait_prior();
  pdl_launch_dependents();
  const int t0 = blockIdx.x * kKV8Rows, hq = blockIdx.y, h = hq / (a.Hq / a.c.Hkv), tid = threadIdx.x;
  const int n = min(kKV8Rows, a.T - t0);
  for (int i = tid; i < n * D; i += 128)
    s->q[i / D][i % D] = __bfloat162float(a.q[(t0 + i / D) * a.ldq + hq * D + i % D]) * a.sl2;
  float acc[kKV8Rows][ND];
  attend_rows<D, FP8>(a.c, a.slot, h, a.p0 + a.T, n, [&](int r) { return a.p0 + t0 + r + 1; }, s, acc);
#pragma unroll
  for (int r = 0; r < kKV8Rows; ++r)
#pragma unroll
    for (int i = 0; i < ND; ++i) {
      const int d = tid + 128 * i;
      if (r >= n || d >= D) continue;
      float o = acc[r][i];
      if (a.gate) o = o / (1.f + __expf(-__bfloat162float(a.gate[(t0 + r) * a.ldg_t + hq * a.ldg_h + d])));
      a.o[(t0 + r) * a.ldo + hq * D + d] = __float2bfloat16(o);
    }
}

cudaError_t attn_prefill_kv8_launch(const AttnPrefillKV8Args& a, cudaStream_t st) {
  cudaError_t e = cudaSuccess;
  kv8_dispatch(a.c.D, a.c.fp8, [&](auto d, auto fp8) {
    constexpr int DD = decltype(d)::value;
    auto k = attn_prefill_kv8_kernel<DD, decltype(fp8)::value>;
    const size_t smem = sizeof(KV8RowsSmem<DD>);
    e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e == cudaSuccess) e = hx_launch_pdl(k, dim3((unsigned)((a.T + kKV8Rows - 1) / kKV8Rows), (unsigned)a.Hq), dim3(128), smem, st, a);
  });
  return e;
}

}  // namespace hx
