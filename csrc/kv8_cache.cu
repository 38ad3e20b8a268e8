// Writing the 8-bit KV cache (kv8.cuh) and reading it back.
//
//   kv8_append  T tokens of one slot from position p0: every block they complete is quantised
//               from its 32 bf16 rows (the earlier ones come from the tail), and the rows of
//               the sequence's last block go to the tail;
//   kv8_read    rows of a slot as bf16: code * scale rounded once, tail rows as they are.
//
// Both are copies with a reduction over 32 x D values in between: bound by bytes. A CTA of 128
// threads takes one block of one kv head, of K or of V, and keeps it in registers between the
// maximum and the codes, so each value is read once.
#include "kv8.cuh"

namespace hx {

// One block of one head: grid (blocks, Hkv, 2), z = 0 for K and 1 for V. Piece i of a thread
// is 16 dims of one key: for K, four neighbouring lanes hold the 64 dims of a panel's row;
// for V, a warp holds the same dims of the 32 keys, so that their codes, written to shared
// memory a byte each, become rows of 32 keys.
template <int D, bool FP8>
__global__ void __launch_bounds__(128) kv8_append_kernel(KV8AppendArgs a) {
  constexpr int NP = D / 64;  // pieces of a thread: 32 x D / 16 / 128
  __shared__ float red[4];
  __shared__ __align__(16) uint8_t vcode[D * kKV8Block];
  pdl_wait_prior();
  pdl_launch_dependents();
  const int b = a.b0 + blockIdx.x, h = blockIdx.y, tid = threadIdx.x;
  const bool isv = blockIdx.z != 0;
  const int L = a.p0 + a.T, j0 = b * kKV8Block;
  const bool whole = j0 + kKV8Block <= L;
  const long long hd = a.c.head(a.slot, h);
  const __nv_bfloat16* src = isv ? a.v + h * a.v_head : a.k + h * a.k_head;
  const long long ld = isv ? a.v_row : a.k_row;
  __nv_bfloat16* tail = (isv ? a.c.vt : a.c.kt) + hd * (NP * kKV8Panel);
  if (whole) {
    float f[NP][16];
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      // K: 8 keys x 4 pieces of a panel to a warp; V: 32 keys x 1 piece
      const int key = isv ? (tid & 31) : ((tid >> 5) * 8 + ((tid & 31) >> 2));
      const int d0 = isv ? (i * 4 + (tid >> 5)) * 16 : i * 64 + (tid & 3) * 16;
      const int j = j0 + key;
      if (j >= a.p0) {
        load16(src + (j - a.p0) * ld, d0, a.vec, f[i]);
      } else if (!isv) {
        load16(tail + ((d0 >> 6) * kKV8Block + key) * 64 + (d0 & 63), 0, 1, f[i]);
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) f[i][e] = __bfloat162float(tail[(d0 + e) * kKV8Block + key]);
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) m = fmaxf(m, kv8_mag(f[i][e]));
    }
    m = warp_max(m);
    if ((tid & 31) == 0) red[tid >> 5] = m;
    __syncthreads();
    m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float inv = kv8_inv<FP8>(m);
    uint8_t* dst = (isv ? a.c.vc : a.c.kc) + a.c.block(a.slot, h, b) * (NP * kKV8Panel);
    if (tid == 0) (isv ? a.c.vs : a.c.ks)[a.c.block(a.slot, h, b)] = kv8_scale<FP8>(m);
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      if (!isv) {
        const int key = (tid >> 5) * 8 + ((tid & 31) >> 2);
        *reinterpret_cast<uint4*>(dst + (i * kKV8Block + key) * 64 + (tid & 3) * 16) =
            make_uint4(kv8_code4<FP8>(f[i], inv), kv8_code4<FP8>(f[i] + 4, inv), kv8_code4<FP8>(f[i] + 8, inv),
                       kv8_code4<FP8>(f[i] + 12, inv));
      } else {
        const int d0 = (i * 4 + (tid >> 5)) * 16;
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const uint32_t q = kv8_code4<FP8>(f[i] + e, inv);
#pragma unroll
          for (int c = 0; c < 4; ++c) vcode[(d0 + e + c) * kKV8Block + (tid & 31)] = (uint8_t)(q >> 8 * c);
        }
      }
    }
    __syncthreads();
    if (isv)
      for (int i = tid; i < D * kKV8Block / 16; i += 128)
        reinterpret_cast<uint4*>(dst)[i] = reinterpret_cast<const uint4*>(vcode)[i];
  }
  // The first block's CTA alone has read the old tail (above), so it writes the new one: the
  // new rows of the sequence's last block.
  if (blockIdx.x != 0) return;
  __syncthreads();
  const int l0 = (L - 1) / kKV8Block * kKV8Block;
  const int r0 = max(a.p0 - l0, 0), rows = L - l0 - r0;
  for (int i = tid; i < rows * (D / 16); i += 128) {
    const int r = r0 + (isv ? i % rows : i / (D / 16));
    const int d0 = (isv ? i / rows : i % (D / 16)) * 16;
    float f[16];
    load16(src + (l0 + r - a.p0) * ld, d0, a.vec, f);
    if (!isv) {
      bf16x8* p = reinterpret_cast<bf16x8*>(tail + ((d0 >> 6) * kKV8Block + r) * 64 + (d0 & 63));
      p[0] = pack8(f);
      p[1] = pack8(f + 8);
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) tail[(d0 + e) * kKV8Block + r] = __float2bfloat16(f[e]);
    }
  }
}

// Grid (blocks, Hkv, 2) of 128 threads as in the append; a thread writes 32 bytes of a row.
template <int D, bool FP8>
__global__ void __launch_bounds__(128) kv8_read_kernel(KV8ReadArgs a) {
  constexpr int NP = D / 64;
  __shared__ __align__(16) uint8_t vcode[D * kKV8Block];
  pdl_wait_prior();
  pdl_launch_dependents();
  const int b = a.start / kKV8Block + blockIdx.x, h = blockIdx.y, tid = threadIdx.x;
  const bool isv = blockIdx.z != 0;
  const int j0 = b * kKV8Block;
  const bool whole = j0 + kKV8Block <= a.L;
  const long long blk = a.c.block(a.slot, h, b);
  const uint8_t* codes = (isv ? a.c.vc : a.c.kc) + blk * (NP * kKV8Panel);
  const __nv_bfloat16* tail = (isv ? a.c.vt : a.c.kt) + a.c.head(a.slot, h) * (NP * kKV8Panel);
  const float scale = whole ? (isv ? a.c.vs : a.c.ks)[blk] : 0.f;
  if (isv && whole) {
    for (int i = tid; i < D * kKV8Block / 16; i += 128)
      reinterpret_cast<uint4*>(vcode)[i] = reinterpret_cast<const uint4*>(codes)[i];
    __syncthreads();
  }
  __nv_bfloat16* out = isv ? a.v + h * a.v_head : a.k + h * a.k_head;
  const long long ld = isv ? a.v_row : a.k_row;
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int key = isv ? (tid & 31) : ((tid >> 5) * 8 + ((tid & 31) >> 2));
    const int d0 = isv ? (i * 4 + (tid >> 5)) * 16 : i * 64 + (tid & 3) * 16;
    const int j = j0 + key;
    if (j < a.start || j >= a.start + a.n) continue;
    float f[16];
    if (!whole) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int d = d0 + e;
        f[e] = __bfloat162float(isv ? tail[d * kKV8Block + key]
                                    : tail[((d >> 6) * kKV8Block + key) * 64 + (d & 63)]);
      }
    } else if (isv) {
#pragma unroll
      for (int e = 0; e < 16; ++e) f[e] = kv8_float<FP8>(vcode[(d0 + e) * kKV8Block + key]) * scale;
    } else {
      const uint4 w = *reinterpret_cast<const uint4*>(codes + (i * kKV8Block + key) * 64 + (tid & 3) * 16);
      const uint8_t* q = reinterpret_cast<const uint8_t*>(&w);
#pragma unroll
      for (int e = 0; e < 16; ++e) f[e] = kv8_float<FP8>(q[e]) * scale;
    }
    bf16x8* p = reinterpret_cast<bf16x8*>(out + (long long)(j - a.start) * ld + d0);
    p[0] = pack8(f);
    p[1] = pack8(f + 8);
  }
}

cudaError_t kv8_append_launch(const KV8AppendArgs& a, cudaStream_t st) {
  const dim3 grid((unsigned)((a.p0 + a.T - 1) / kKV8Block - a.b0 + 1), (unsigned)a.c.Hkv, 2);
  cudaError_t e = cudaSuccess;
  kv8_dispatch(a.c.D, a.c.fp8, [&](auto d, auto fp8) {
    e = hx_launch_pdl(kv8_append_kernel<decltype(d)::value, decltype(fp8)::value>, grid, dim3(128), 0, st, a);
  });
  return e;
}

cudaError_t kv8_read_launch(const KV8ReadArgs& a, cudaStream_t st) {
  const dim3 grid((unsigned)((a.start + a.n - 1) / kKV8Block - a.start / kKV8Block + 1), (unsigned)a.c.Hkv, 2);
  cudaError_t e = cudaSuccess;
  kv8_dispatch(a.c.D, a.c.fp8, [&](auto d, auto fp8) {
    e = hx_launch_pdl(kv8_read_kernel<decltype(d)::value, decltype(fp8)::value>, grid, dim3(128), 0, st, a);
  });
  return e;
}

}  // namespace hx
