// Attention of up to 16 query rows that share a kv head over the 8-bit KV cache: the softmax
// over one block of 32 keys at a time, in f32.
#pragma once
#include "kv8.cuh"

namespace hx {

constexpr int kKV8Rows = 16;

template <int D>
struct KV8RowsSmem {
  float q[kKV8Rows][D];
  float k[kKV8Block][D + 1];
  float v[kKV8Block][D];
  float s[kKV8Rows][kKV8Block];
  float m[kKV8Rows], l[kKV8Rows], f[kKV8Rows];
};

// Rows q[0 .. n) of s (scaled by scale * log2 e) attend to keys 0 .. lim(row) - 1 of a slot with L tokens;
// 128 threads. acc[r][i] is output dim tid + 128 i of row r (0 where a row has no key).
template <int D, bool FP8, typename Lim>
HX_DEVICE void attend_rows(const KV8& c, int slot, int h, int L, int n, Lim lim, KV8RowsSmem<D>* s,
                           float (&acc)[kKV8Rows][(D + 127) / 128]) {
  constexpr int ND = (D + 127) / 128;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid < kKV8Rows) { s->m[tid] = -INFINITY; s->l[tid] = 0.f; }
#pragma unroll
  for (int r = 0; r < kKV8Rows; ++r)
#pragma unroll
    for (int i = 0; i < ND; ++i) acc[r][i] = 0.f;
  int kend = 0;
  for (int r = 0; r < n; ++r) kend = max(kend, lim(r));
#pragma unroll 1
  for (int b = 0; b * kKV8Block < kend; ++b) {
    const bool whole = (b + 1) * kKV8Block <= L;
    const long long blk = c.block(slot, h, b), base = blk * (D * kKV8Block);
    const long long tbase = c.head(slot, h) * (D * kKV8Block);
    const float ks = whole ? c.ks[blk] : 1.f, vs = whole ? c.vs[blk] : 1.f;
    __syncthreads();
#pragma unroll 1
    for (int i = tid; i < D * kKV8Block; i += 128) {
      const int p = i / kKV8Panel, w = i % kKV8Panel;  // panel, place in it
      const int kk = w / 64, kd = p * 64 + w % 64, vd = p * 64 + w / 32, vk = w % 32;
      const bool in_k = b * kKV8Block + kk < L, in_v = b * kKV8Block + vk < L;  // the tail's other rows hold anything
      s->k[kk][kd] = !in_k ? 0.f : whole ? kv8_float<FP8>(c.kc[base + i]) * ks : __bfloat162float(c.kt[tbase + i]);
      s->v[vk][vd] = !in_v ? 0.f : whole ? kv8_float<FP8>(c.vc[base + i]) * vs : __bfloat162float(c.vt[tbase + i]);
    }
    __syncthreads();
    for (int r = warp; r < n; r += 4) {
      float x = 0.f;
#pragma unroll 4
      for (int d = 0; d < D; ++d) x += s->q[r][d] * s->k[lane][d];
      if (b * kKV8Block + lane >= lim(r)) x = -INFINITY;
      const float mo = s->m[r], mn = fmaxf(mo, warp_max(x));
      const float p = x == -INFINITY ? 0.f : exp2f(x - mn);
      const float ps = warp_sum(p);
      s->s[r][lane] = p;
      __syncwarp();
      if (lane == 0) {
        const float f = mo == -INFINITY ? 0.f : exp2f(mo - mn);
        s->f[r] = f;
        s->l[r] = s->l[r] * f + ps;
        s->m[r] = mn;
      }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kKV8Rows; ++r) {
      if (r >= n) break;
#pragma unroll
      for (int i = 0; i < ND; ++i) {
        const int d = tid + 128 * i;
        if (d >= D) continue;
        float o = acc[r][i] * s->f[r];
#pragma unroll 2
        for (int j = 0; j < kKV8Block; ++j) o = fmaf(s->s[r][j], s->v[j][d], o);
        acc[r][i] = o;
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kKV8Rows; ++r)
    if (r < n) {
      const float inv = s->l[r] > 0.f ? 1.f / s->l[r] : 0.f;
#pragma unroll
      for (int i = 0; i < ND; ++i) acc[r][i] *= inv;
    }
}

}  // namespace hx
