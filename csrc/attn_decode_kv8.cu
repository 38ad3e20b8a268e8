// Single-token GQA attention over the 8-bit KV cache (kv8.cuh), with the work around it in the
// same launch: q / k RMSNorm per head, rotate-half RoPE, the append of the new token (and the
// quantisation of the block that it completes), softmax attention over [0, pos] and the
// sigmoid output gate. Arguments as attn_decode.
//
//   s_j = (q . c_j) * ks_b * scale,  o = sum_b vs_b sum_{j in b} p_j c'_j / sum_j p_j
// for codes c (K) and c' (V) of block b: the codes are exact in f16, so both products run on the
// tensor cores over codes, and the scales are f32 factors outside them.
//
// Work is laid out as one list of blocks (32 keys of one sequence and kv head) over the whole
// ragged batch. Clusters of kCL CTAs take equal runs of it, so sequences of any mix of lengths
// load every SM alike; a run may end inside a pair (sequence, kv head) and go on into the next.
// Inside a run's part of one pair (a segment) every warp of the cluster takes whole blocks, a
// warp with its own ring of bulk copies: K and V blocks are contiguous panels, so a copy is one
// 2 or 4 KB piece and no warp waits for another. The warps' (max, sum, O) merge through shared
// memory, the CTAs' through distributed shared memory, and segments of one pair through global
// scratch, merged by the cluster that finishes last.
//
// q and k stay in f32 between the norm, the rotation and the products; K is rounded to bf16
// once, as it enters the cache. q enters the products in f16 after a power of two that brings
// its largest entry to 128..256 (11 bits; entries 2^32 below the largest vanish), p in f16 as
// 256 * exp(s - max). The incomplete last block is bf16 and may hold any exponent: its products
// are bf16 ones on q and p split into two bf16 parts (16 bits).
#include <cooperative_groups.h>

#include "kv8.cuh"
#include "mma_frag.cuh"
#include "tc_common.cuh"

namespace cg = cooperative_groups;

namespace hx {

constexpr int kKV8Warps = 4;   // warps of a CTA

template <int D>
struct KV8Ring {
  static constexpr int kUnit = (D >= 128 ? 128 : D) * kKV8Block;  // bytes of a copy
  static constexpr int kUK = D * kKV8Block / kUnit;               // copies of a K (or V) block
  static constexpr int kSlots = D >= 128 ? 6 : 8;                 // slots of a warp's ring
};

template <int D, int NT>
struct DecodeKV8Smem {
  static constexpr int GP = NT * 8;      // heads of a pass, padded
  static constexpr int LD = D + 4;       // row stride of wo: lanes of one store hit distinct banks
  union {
    alignas(128) uint8_t ring[kKV8Warps][KV8Ring<D>::kSlots][KV8Ring<D>::kUnit];
    float wo[kKV8Warps][GP][LD];         // the warps' O, then (in [0]) the CTA's
  };
  float q[GP][D];                        // normed, rotated, times a power of two
  float kn[D];                           // the new token's key
  float cs[D / 2], sn[D / 2];            // rotation of the sequence's position
  alignas(16) __nv_bfloat16 knew[D], vnew[D];        // the new token as the cache holds it
  float qmul[GP];                        // score factor of each head: scale * log2(e) / power of two
  float wm[kKV8Warps][GP], wl[kKV8Warps][GP];
  float cm[GP], cl[GP];                  // this CTA's (max, sum)
  float pw[GP][kKV8CL];                  // the cluster's CTAs' weights
  float fw[GP][kKV8MaxPart];             // the partials' weights in the last merge
  uint64_t full[kKV8Warps][KV8Ring<D>::kSlots];
  int off[kKV8MaxBatch + 1];             // blocks before sequence b
  float red[2][kKV8Warps];
  int last;
};

HX_DEVICE void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

HX_DEVICE uint32_t movmatrix_t(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

HX_DEVICE void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   tc::smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(tc::smem_u32(bar))
               : "memory");
}

HX_DEVICE uint32_t pack_f16x2(float lo, float hi) {
  __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

// Four codes -> two f16 pairs, exactly. int8: a byte offset by 128 under the exponent of 1024
// is 1024 + code + 128.
template <bool FP8>
HX_DEVICE void codes_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (FP8) {
    const __half2_raw a = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffff), __NV_E4M3);
    const __half2_raw b = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), __NV_E4M3);
    lo = *reinterpret_cast<const uint32_t*>(&a);
    hi = *reinterpret_cast<const uint32_t*>(&b);
  } else {
    const uint32_t u = w ^ 0x80808080u;
    const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    const uint32_t bias = 0x64806480u;  // 1152
    const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&bias));
    const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&b), *reinterpret_cast<const __half2*>(&bias));
    lo = *reinterpret_cast<const uint32_t*>(&x);
    hi = *reinterpret_cast<const uint32_t*>(&y);
  }
}

// The key that row r (0..7) of score tile (s, j) holds. P's tiles then transpose into operands
// whose pairs of keys lie together in V's rows of 32 keys: lane (g, t) reads keys 8t .. 8t+7.
HX_DEVICE int key_of(int s, int j, int r) { return 8 * (r >> 1) + (r & 1) + 4 * s + 2 * j; }

template <int D, int NT, bool FP8>
struct DecodeKV8Warp {
  static constexpr int NP = D / 64;
  uint32_t qb[NT][D / 16][2];   // Q as the B operand
  float mul[NT][2];             // score factors of heads 8 nt + 2 t + e
  float m[NT][2], l[NT][2];     // running max; this lane's part of the running sum
  float acc[D / 16][NT][4];     // O^T: dims 16 i + g (+8), heads 8 nt + 2 t + e
  float sc[2][NT][4];
  uint32_t pb[2][NT][2];
  float corr[NT][2];

  HX_DEVICE void reset() {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) { m[nt][e] = -INFINITY; l[nt][e] = 0.f; }
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[i][nt][c] = 0.f;
  }

  HX_DEVICE void clear_scores() {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 4; ++c) sc[s][nt][c] = 0.f;
  }

  // scores += Q . K over the 64 dims of panel u (32 keys x 64 codes in shared memory)
  HX_DEVICE void qk_panel(const uint8_t* p, int u) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const uint4 x = *reinterpret_cast<const uint4*>(p + key_of(s, 0, g) * 64 + t * 16);
      const uint4 y = *reinterpret_cast<const uint4*>(p + key_of(s, 1, g) * 64 + t * 16);
      const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t a0, a1, a2, a3;
        codes_to_f16<FP8>(xs[k], a0, a2);
        codes_to_f16<FP8>(ys[k], a1, a3);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma_f16(sc[s][nt], a0, a1, a2, a3, qb[nt][u * 4 + k][0], qb[nt][u * 4 + k][1]);
      }
    }
  }

  // O^T += V^T . P over the 64 dims of panel u (64 dims x 32 codes in shared memory)
  HX_DEVICE void pv_panel(const uint8_t* p, int u, float vs) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint2 x = *reinterpret_cast<const uint2*>(p + (i * 16 + g) * 32 + t * 8);
      const uint2 y = *reinterpret_cast<const uint2*>(p + (i * 16 + g + 8) * 32 + t * 8);
      uint32_t a[2][4];
      codes_to_f16<FP8>(x.x, a[0][0], a[0][2]);
      codes_to_f16<FP8>(y.x, a[0][1], a[0][3]);
      codes_to_f16<FP8>(x.y, a[1][0], a[1][2]);
      codes_to_f16<FP8>(y.y, a[1][1], a[1][3]);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < 2; ++s) mma_f16(o, a[s][0], a[s][1], a[s][2], a[s][3], pb[s][nt][0], pb[s][nt][1]);
        float (&c)[4] = acc[u * 4 + i][nt];
#pragma unroll
        for (int e = 0; e < 4; ++e) c[e] = fmaf(c[e], corr[nt][e & 1], o[e] * vs);
      }
    }
  }

  // Scores -> probabilities in sc (256 exp2(s - max)); the running max and sums move on.
  // Keys past `lastkey` are out.
  HX_DEVICE void softmax(float ks, int lastkey) {
    const int g = (threadIdx.x & 31) >> 2;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float f = mul[nt][e] * ks;
        float mx = -INFINITY;
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float& x = sc[s][nt][2 * j + e];
            x = key_of(s, j, g) <= lastkey ? x * f : -INFINITY;
            mx = fmaxf(mx, x);
          }
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const float mn = fmaxf(m[nt][e], mx);
        const float base = mn == -INFINITY ? 0.f : mn - 8.f;
        corr[nt][e] = exp2f(m[nt][e] - mn);
        if (m[nt][e] == -INFINITY) corr[nt][e] = 0.f;
        float sum = 0.f;
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float& x = sc[s][nt][2 * j + e];
            x = exp2f(x - base);
            sum += x;
          }
        l[nt][e] = fmaf(l[nt][e], corr[nt][e], sum);
        m[nt][e] = mn;
      }
  }

  HX_DEVICE void pack_p() {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) pb[s][nt][j] = movmatrix_t(pack_f16x2(sc[s][nt][2 * j], sc[s][nt][2 * j + 1]));
  }
};

// One bf16 operand pair split in two: x = hi + lo to 16 bits.
HX_DEVICE void split_bf16x2(float x, float y, uint32_t& hi, uint32_t& lo) {
  hi = pack_bf16x2(x, y);
  const __nv_bfloat162 h = *reinterpret_cast<const __nv_bfloat162*>(&hi);
  const float2 f = __bfloat1622float2(h);
  lo = pack_bf16x2(x - f.x, y - f.y);
}

template <int D, int NT, bool FP8>
__global__ void __launch_bounds__(kKV8Warps * 32, 2) attn_decode_kv8_kernel(AttnDecodeKV8Args a) {
  using R = KV8Ring<D>;
  using SM = DecodeKV8Smem<D, NT>;
  constexpr int GP = SM::GP, NP = D / 64, NW = kKV8Warps, NTH = NW * 32;
  extern __shared__ __align__(128) unsigned char raw[];
  SM* s = reinterpret_cast<SM*>(raw);
  cg::cluster_group cluster = cg::this_cluster();
  constexpr int CL = kKV8CL;
  const int crank = (int)cluster.block_rank(), cid = blockIdx.x / CL, NC = gridDim.x / CL;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int Hkv = a.c.Hkv, G = a.Hq / Hkv, HG = a.HG, per = (G + HG - 1) / HG, PB = Hkv * HG;
  const int qw = a.gated ? 2 * D : D;
  if (tid == 0) {
    for (int w = 0; w < NW; ++w)
      for (int i = 0; i < R::kSlots; ++i) tc::mbar_init(&s->full[w][i], 1);
    tc::fence_barrier_init();
  }
  pdl_wait_prior();
  pdl_launch_dependents();
  // ---- blocks of each sequence (0: refused), and the blocks before it -------------------------
  if (warp == 0) {
    int base = 0;
    for (int b0 = 0; b0 < a.B; b0 += 32) {
      int n = 0;
      if (b0 + lane < a.B) {
        const int slot = a.slots[b0 + lane];
        const int p = slot >= 0 && slot < a.c.S ? a.pos[slot] : -1;
        n = p >= 0 && p < a.c.nb * kKV8Block ? p / kKV8Block + 1 : 0;
      }
      int x = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      if (b0 + lane < a.B) s->off[b0 + lane + 1] = base + x;
      base += __shfl_sync(0xffffffffu, x, 31);
    }
    if (lane == 0) s->off[0] = 0;
  }
  __syncthreads();
  if (cid == 0 && crank == 0)  // refused sequences: no cache access, a zero row, the error word
    for (int b = 0; b < a.B; ++b)
      if (s->off[b + 1] == s->off[b]) {
        for (int i = tid; i < a.Hq * D; i += NTH) a.out[(long long)b * a.Hq * D + i] = __float2bfloat16(0.f);
        if (tid == 0) atomicCAS(a.ws, 0, 6001);
      }
  // Runs of `chunk` blocks. At least a block for every warp of the cluster where a pair has as
  // many: a pair split further would only add partials to merge.
  const long long W = (long long)s->off[a.B] * PB;
  int nbmax = 0;
  for (int b = 0; b < a.B; ++b) nbmax = max(nbmax, s->off[b + 1] - s->off[b]);
  const long long chunk = max((W + NC - 1) / NC, (long long)min(nbmax, CL * NW));
  long long w = cid * chunk;
  const long long wend = min(W, w + chunk);
  if (w >= wend) return;  // the whole cluster
  float* part_o = reinterpret_cast<float*>(a.ws + kKV8PartAt);  // [NC + pairs][GP][D]
  float* part_ml = part_o + (long long)(NC + a.B * PB) * GP * D;  // [NC + pairs][GP][2]
  unsigned seq = 0;  // copies this warp has issued in all
  bool ok = true;
  DecodeKV8Warp<D, NT, FP8> st;
  int b = 0;
  while (w < wend) {
    while ((long long)s->off[b + 1] * PB <= w) ++b;
    const int nb = s->off[b + 1] - s->off[b];
    const int pl = (int)((w - (long long)s->off[b] * PB) / nb);      // kv head and head group
    const long long p0 = (long long)s->off[b] * PB + (long long)pl * nb;  // the pair's first block in the list
    const int blk0 = (int)(w - p0), blk1 = (int)min((long long)nb, wend - p0);
    const int pair = b * PB + pl, h = pl / HG, hg = pl % HG, g0 = hg * per, n = min(per, G - g0);
    const int slot = a.slots[b], p = a.pos[slot], row = p % kKV8Block;
    const __nv_bfloat16* pr = a.proj + b * a.ldp;
    // ---- this warp's blocks: blk0 + gw, + CL * NW, ...; the sequence's last block is not copied --
    const int gw = crank * NW + warp;
    const int my0 = blk0 + gw;
    const int n8 = min(blk1, nb - 1);
    const int mine = my0 < n8 ? (n8 - my0 + CL * NW - 1) / (CL * NW) : 0;  // complete blocks
    const bool has_last = blk1 == nb && (nb - 1 - blk0) % (CL * NW) == gw;
    const bool cta_last = blk1 == nb && (nb - 1 - blk0) % (CL * NW) / NW == crank;
    const unsigned units = (unsigned)mine * 2 * R::kUK;
    const uint8_t* kbase = a.c.kc + a.c.block(slot, h, 0) * (D * kKV8Block);
    const uint8_t* vbase = a.c.vc + a.c.block(slot, h, 0) * (D * kKV8Block);
    auto issue = [&](unsigned i) {  // lane 0: unit i of this segment
      const unsigned sl = (seq + i) % R::kSlots, in = i % (2 * R::kUK);
      const long long blk = my0 + (long long)(i / (2 * R::kUK)) * (CL * NW);
      const uint8_t* src = (in < R::kUK ? kbase : vbase) + blk * (D * kKV8Block) + (in % R::kUK) * R::kUnit;
      tc::mbar_expect_tx(&s->full[warp][sl], R::kUnit);
      bulk_load(s->ring[warp][sl], src, R::kUnit, &s->full[warp][sl]);
    };
    // (the warp with the last block starts its copies after it: the block's codes may be made in
    // its ring)
    if (lane == 0 && ok && !has_last)
      for (unsigned i = 0; i < min(units, (unsigned)R::kSlots); ++i) issue(i);
    // ---- q of the group's heads (and the new key): norm, rotation ------------------------------
    const int prot = p + (a.rope_delta ? a.rope_delta[slot] : 0);
    for (int i = tid; i < a.rot / 2; i += NTH) sincosf((float)prot * a.inv_freq[i], &s->sn[i], &s->cs[i]);
    __syncthreads();
    for (int r = warp; r < n + (cta_last ? 1 : 0); r += NW) {
      const bool isk = r == n;
      const __nv_bfloat16* src = isk ? pr + a.Hq * qw + h * D : pr + (long long)(h * G + g0 + r) * qw;
      const float* nw = isk ? a.k_norm_w : a.q_norm_w;
      float* x = isk ? s->kn : s->q[r];
      float v[D / 32];
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        v[i] = __bfloat162float(src[i * 32 + lane]);
        ss += v[i] * v[i];
      }
      if (nw) {
        const float inv = rsqrtf(warp_sum(ss) / D + a.eps);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) v[i] *= inv * nw[i * 32 + lane];
      }
#pragma unroll
      for (int i = 0; i < D / 32; ++i) x[i * 32 + lane] = v[i];
      __syncwarp();
      const int half = a.rot / 2;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        const int d = i * 32 + lane;
        if (d < a.rot) v[i] = d < half ? v[i] * s->cs[d] - x[d + half] * s->sn[d]
                                       : v[i] * s->cs[d - half] + x[d - half] * s->sn[d - half];
      }
      __syncwarp();
      if (isk) {
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          const int d = i * 32 + lane;
          s->knew[d] = __float2bfloat16(v[i]);
          s->vnew[d] = pr[a.Hq * qw + (Hkv + h) * D + d];
        }
      } else {
        float mag = 0.f;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) mag = fmaxf(mag, kv8_mag(v[i]));
        mag = warp_max(mag);
        // power of two that brings the largest entry to 128..256
        const int ex = min(134 - (int)(__float_as_uint(mag) >> 23), 120);
        const float up = __uint_as_float((uint32_t)(ex + 127) << 23);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) x[i * 32 + lane] = v[i] * up;
        if (lane == 0) s->qmul[r] = a.sl2 / up;
      }
    }
    __syncthreads();
    if (cta_last && hg == 0) {  // the new token enters the tail
      __nv_bfloat16* kt = a.c.kt + a.c.head(slot, h) * (NP * kKV8Panel);
      __nv_bfloat16* vt = a.c.vt + a.c.head(slot, h) * (NP * kKV8Panel);
      for (int d = tid; d < D; d += NTH) {
        kt[((d >> 6) * kKV8Block + row) * 64 + (d & 63)] = s->knew[d];
        vt[d * kKV8Block + row] = s->vnew[d];
      }
    }
    // A block that this token completes gets its codes: into the ring of the warp that attends to
    // it and into the cache. Every head group derives them; the first one stores them.
    const bool completes = cta_last && row == kKV8Block - 1;
    uint8_t* fresh = s->ring[(nb - 1 - blk0) % NW][0];  // that warp's ring, not in use yet
    float scale[2];
    if (completes) {
      uint4 x[2][NP][2];
      float mag[2] = {0.f, 0.f};
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        const __nv_bfloat16* src = (z ? a.c.vt : a.c.kt) + a.c.head(slot, h) * (NP * kKV8Panel);
#pragma unroll
        for (int i = 0; i < NP; ++i) {  // 16 values from c * 16 on of the block's layout
          const int c = i * NTH + tid;
          x[z][i][0] = *reinterpret_cast<const uint4*>(src + c * 16);
          x[z][i][1] = *reinterpret_cast<const uint4*>(src + c * 16 + 8);
          if (z) {
            if (c & 1)  // key 31 of dim c / 2
              x[z][i][1].w = (x[z][i][1].w & 0xffffu) | (uint32_t)__bfloat16_as_ushort(s->vnew[c >> 1]) << 16;
          } else if ((c & 127) >= 124) {  // key 31 of panel c / 128
            const uint4* kn = reinterpret_cast<const uint4*>(s->knew + (c >> 7) * 64 + (c & 3) * 16);
            x[z][i][0] = kn[0];
            x[z][i][1] = kn[1];
          }
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            float f[8];
            unpack8(*reinterpret_cast<const bf16x8*>(&x[z][i][q]), f);
#pragma unroll
            for (int e = 0; e < 8; ++e) mag[z] = fmaxf(mag[z], kv8_mag(f[e]));
          }
        }
        mag[z] = warp_max(mag[z]);
        if (lane == 0) s->red[z][warp] = mag[z];
      }
      __syncthreads();
      const long long at = a.c.block(slot, h, nb - 1);
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        const float m = fmaxf(fmaxf(s->red[z][0], s->red[z][1]), fmaxf(s->red[z][2], s->red[z][3]));
        const float inv = kv8_inv<FP8>(m);
        scale[z] = kv8_scale<FP8>(m);
        uint8_t* dst = (z ? a.c.vc : a.c.kc) + at * (D * kKV8Block);
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          float f[16];
          unpack8(*reinterpret_cast<const bf16x8*>(&x[z][i][0]), f);
          unpack8(*reinterpret_cast<const bf16x8*>(&x[z][i][1]), f + 8);
          const uint4 v = make_uint4(kv8_code4<FP8>(f, inv), kv8_code4<FP8>(f + 4, inv), kv8_code4<FP8>(f + 8, inv),
                                     kv8_code4<FP8>(f + 12, inv));
          reinterpret_cast<uint4*>(fresh + z * D * kKV8Block)[i * NTH + tid] = v;
          if (hg == 0) reinterpret_cast<uint4*>(dst)[i * NTH + tid] = v;
        }
        if (hg == 0 && tid == 0) (z ? a.c.vs : a.c.ks)[at] = scale[z];
      }
      __syncthreads();
    }
    st.reset();
    if (mine > 0 || has_last) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const bool in = nt * 8 + g < n;
        const float* q = s->q[nt * 8 + g];
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const int d = (k >> 2) * 64 + t * 16 + (k & 3) * 4;
          const float4 x = *reinterpret_cast<const float4*>(q + d);
          st.qb[nt][k][0] = in ? pack_f16x2(x.x, x.y) : 0u;
          st.qb[nt][k][1] = in ? pack_f16x2(x.z, x.w) : 0u;
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) st.mul[nt][e] = nt * 8 + 2 * t + e < n ? s->qmul[nt * 8 + 2 * t + e] : 0.f;
      }
    }
    // ---- the sequence's last block: bf16 rows of the tail and the new token ----------------------
    if (has_last) {
      const __nv_bfloat16* kt = a.c.kt + a.c.head(slot, h) * (NP * kKV8Panel);
      const __nv_bfloat16* vt = a.c.vt + a.c.head(slot, h) * (NP * kKV8Panel);
      if (completes) {
        st.clear_scores();
#pragma unroll
        for (int q = 0; q < NP; ++q) st.qk_panel(fresh + q * kKV8Panel, q);
        st.softmax(scale[0], kKV8Block);
        st.pack_p();
#pragma unroll
        for (int q = 0; q < NP; ++q) st.pv_panel(fresh + D * kKV8Block + q * kKV8Panel, q, scale[1]);
      } else {
        st.clear_scores();
#pragma unroll 1
        for (int pn = 0; pn < NP; ++pn)
#pragma unroll
          for (int sx = 0; sx < 2; ++sx) {
            uint32_t kx[2][8];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              // rows past the new token hold anything: their scores are replaced in softmax()
              const int key = key_of(sx, j, g);
              const __nv_bfloat16* r = key == row ? s->knew + pn * 64 : kt + (pn * kKV8Block + key) * 64;
              const uint4 x = *reinterpret_cast<const uint4*>(r + t * 16);
              const uint4 y = *reinterpret_cast<const uint4*>(r + t * 16 + 8);
              kx[j][0] = x.x; kx[j][1] = x.y; kx[j][2] = x.z; kx[j][3] = x.w;
              kx[j][4] = y.x; kx[j][5] = y.y; kx[j][6] = y.z; kx[j][7] = y.w;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                const int hr = nt * 8 + g;
                float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
                if (hr < n) x = *reinterpret_cast<const float4*>(s->q[hr] + pn * 64 + t * 16 + k * 4);
                uint32_t h0, l0, h1, l1;
                split_bf16x2(x.x, x.y, h0, l0);
                split_bf16x2(x.z, x.w, h1, l1);
                mma_16816(st.sc[sx][nt], kx[0][2 * k], kx[1][2 * k], kx[0][2 * k + 1], kx[1][2 * k + 1], h0, h1);
                mma_16816(st.sc[sx][nt], kx[0][2 * k], kx[1][2 * k], kx[0][2 * k + 1], kx[1][2 * k + 1], l0, l1);
              }
          }
        st.softmax(1.f, row);
        uint32_t ph[2][NT][2], plo[2][NT][2];
#pragma unroll
        for (int sx = 0; sx < 2; ++sx)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              uint32_t hi, lo;
              split_bf16x2(st.sc[sx][nt][2 * j], st.sc[sx][nt][2 * j + 1], hi, lo);
              ph[sx][nt][j] = movmatrix_t(hi);
              plo[sx][nt][j] = movmatrix_t(lo);
            }
        // keys 8t .. 8t+7 of a dim: the new token's value goes in, keys past it are cleared
        // (a probability of zero does not silence an infinity or a NaN)
        auto vload = [&](int d, uint32_t (&x)[4]) {
          const uint4 v = *reinterpret_cast<const uint4*>(vt + d * kKV8Block + t * 8);
          x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
          const uint32_t nv = __bfloat16_as_ushort(s->vnew[d]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = t * 8 + e * 2;
            if (key == row) x[e] = nv;
            else if (key + 1 == row) x[e] = (x[e] & 0xffffu) | nv << 16;
            else if (key > row) x[e] = 0u;
          }
        };
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          uint32_t x[4], y[4];
          vload(i * 16 + g, x);
          vload(i * 16 + g + 8, y);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int sx = 0; sx < 2; ++sx) {
              mma_16816(o, x[2 * sx], y[2 * sx], x[2 * sx + 1], y[2 * sx + 1], ph[sx][nt][0], ph[sx][nt][1]);
              mma_16816(o, x[2 * sx], y[2 * sx], x[2 * sx + 1], y[2 * sx + 1], plo[sx][nt][0], plo[sx][nt][1]);
            }
            float (&c)[4] = st.acc[i][nt];
#pragma unroll
            for (int e = 0; e < 4; ++e) c[e] = fmaf(c[e], st.corr[nt][e & 1], o[e]);
          }
        }
      }
      if (completes) tc::fence_proxy_async_smem();  // codes in the ring before copies into it
      __syncwarp();
      if (lane == 0 && ok)
        for (unsigned i = 0; i < min(units, (unsigned)R::kSlots); ++i) issue(i);
    }
    // ---- complete blocks -----------------------------------------------------------------------
    const float* ksp = a.c.ks + a.c.block(slot, h, 0);
    const float* vsp = a.c.vs + a.c.block(slot, h, 0);
    unsigned u = 0;
    auto next_unit = [&](auto&& use) {  // wait for unit u, use it, hand its slot to unit u + kSlots
      const unsigned sl = (seq + u) % R::kSlots;
      if (ok) ok = tc::mbar_wait(&s->full[warp][sl], ((seq + u) / R::kSlots) & 1, a.ws, 6002);
      ok = __all_sync(0xffffffffu, ok);
      use(s->ring[warp][sl]);
      __syncwarp();
      if (lane == 0 && ok && u + R::kSlots < units) issue(u + R::kSlots);
      ++u;
    };
    for (int i = 0; i < mine && ok; ++i) {
      const int blk = my0 + i * (CL * NW);
      const float ks = __ldcg(ksp + blk), vs = __ldcg(vsp + blk);
      st.clear_scores();
#pragma unroll
      for (int k = 0; k < R::kUK; ++k)
        next_unit([&](const uint8_t* x) {
#pragma unroll
          for (int q = 0; q < R::kUnit / kKV8Panel; ++q) st.qk_panel(x + q * kKV8Panel, k * (R::kUnit / kKV8Panel) + q);
        });
      st.softmax(ks, kKV8Block);
      st.pack_p();
#pragma unroll
      for (int k = 0; k < R::kUK; ++k)
        next_unit([&](const uint8_t* x) {
#pragma unroll
          for (int q = 0; q < R::kUnit / kKV8Panel; ++q)
            st.pv_panel(x + q * kKV8Panel, k * (R::kUnit / kKV8Panel) + q, vs);
        });
    }
    seq += units;
    // ---- merge the warps: the ring's memory holds their O now --------------------------------------
    __syncthreads();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float x = st.l[nt][e];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
        if (g == 0) {
          s->wm[warp][nt * 8 + 2 * t + e] = st.m[nt][e];
          s->wl[warp][nt * 8 + 2 * t + e] = x;
        }
      }
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 4; ++c) s->wo[warp][nt * 8 + 2 * t + (c & 1)][i * 16 + g + (c >> 1) * 8] = st.acc[i][nt][c];
    __syncthreads();
    for (int i = tid; i < n * D; i += NTH) {
      const int r = i / D, d = i % D;
      float M = -INFINITY;
#pragma unroll
      for (int x = 0; x < NW; ++x) M = fmaxf(M, s->wm[x][r]);
      float O = 0.f, L = 0.f;
      if (M != -INFINITY)
#pragma unroll
        for (int x = 0; x < NW; ++x) {
          const float f = exp2f(s->wm[x][r] - M);
          O = fmaf(s->wo[x][r][d], f, O);
          L = fmaf(s->wl[x][r], f, L);
        }
      s->wo[0][r][d] = O;  // this thread alone reads and writes (r, d)
      if (d == 0) { s->cm[r] = M; s->cl[r] = L; }
    }
    // ---- merge the cluster's CTAs: each finishes 1 / CL of the columns -------------------
    cluster.sync();
    if (tid < n) {
      float m[CL], M = -INFINITY, L = 0.f;
#pragma unroll
      for (int x = 0; x < CL; ++x) {
        m[x] = *cluster.map_shared_rank(&s->cm[tid], x);
        M = fmaxf(M, m[x]);
      }
#pragma unroll
      for (int x = 0; x < CL; ++x) {
        const float f = m[x] == -INFINITY ? 0.f : exp2f(m[x] - M);
        L = fmaf(*cluster.map_shared_rank(&s->cl[tid], x), f, L);
        s->pw[tid][x] = f;
      }
      s->wm[0][tid] = M;
      s->wl[0][tid] = L;
    }
    __syncthreads();
    auto finish = [&](int r, int d, float o) {  // o: the row's output
      const int hq = h * G + g0 + r;
      if (a.gated) o = o / (1.f + __expf(-__bfloat162float(pr[(long long)hq * qw + D + d])));
      a.out[((long long)b * a.Hq + hq) * D + d] = __float2bfloat16(o);
    };
    const bool alone = blk0 == 0 && blk1 == nb;
    const int cols = n * D / CL;
    const long long at = (cid + pair) * (long long)(GP * D);
    for (int i = crank * cols + tid; i < (crank + 1) * cols; i += NTH) {
      const int r = i / D, d = i % D;
      float O = 0.f;
#pragma unroll
      for (int x = 0; x < CL; ++x) O = fmaf(cluster.map_shared_rank(&s->wo[0][r][0], x)[d], s->pw[r][x], O);
      if (alone) finish(r, d, O / s->wl[0][r]);
      else part_o[at + i] = O;
    }
    if (!alone) {
      if (crank == 0 && tid < n) {
        part_ml[((long long)(cid + pair) * GP + tid) * 2] = s->wm[0][tid];
        part_ml[((long long)(cid + pair) * GP + tid) * 2 + 1] = s->wl[0][tid];
      }
      __threadfence();
    }
    tc::fence_proxy_async_smem();  // O's stores before the next segment's copies into the same memory
    cluster.sync();
    if (!alone) {
      // the cluster that completes the pair's block count merges its partials
      if (crank == 0 && tid == 0) {
        int* counter = a.ws + kKV8Err + pair;
        const int done = atomicAdd(counter, blk1 - blk0) + (blk1 - blk0);
        if (done == nb) *counter = 0;
        const int last = done == nb;
        for (int x = 0; x < CL; ++x) *cluster.map_shared_rank(&s->last, x) = last;
        __threadfence();
      }
      cluster.sync();
      if (s->last) {
        __threadfence();
        const int c0 = (int)(p0 / chunk), np = (int)((p0 + nb - 1) / chunk) - c0 + 1;  // its clusters
        for (int r = warp; r < n; r += NW) {
          float M = -INFINITY;
          for (int x = lane; x < np; x += 32) M = fmaxf(M, __ldcg(&part_ml[((long long)(c0 + x + pair) * GP + r) * 2]));
          M = warp_max(M);
          float L = 0.f;
          for (int x = lane; x < np; x += 32) {
            const long long j = ((long long)(c0 + x + pair) * GP + r) * 2;
            const float f = exp2f(__ldcg(&part_ml[j]) - M);
            L = fmaf(__ldcg(&part_ml[j + 1]), f, L);
            s->fw[r][x] = f;
          }
          L = warp_sum(L);
          if (lane == 0) s->wl[0][r] = L;
        }
        __syncthreads();
        for (int i = crank * cols + tid; i < (crank + 1) * cols; i += NTH) {
          const int r = i / D, d = i % D;
          float O = 0.f;
#pragma unroll 8
          for (int x = 0; x < np; ++x)
            O = fmaf(__ldcg(&part_o[(long long)(c0 + x + pair) * (GP * D) + i]), s->fw[r][x], O);
          finish(r, d, O / s->wl[0][r]);
        }
        __syncthreads();
      }
    }
    w = p0 + blk1;
  }
}

template <int D, int NT, bool FP8>
static cudaError_t launch_decode(const AttnDecodeKV8Args& a, cudaStream_t st) {
  auto k = attn_decode_kv8_kernel<D, NT, FP8>;
  const size_t smem = sizeof(DecodeKV8Smem<D, NT>);
  static_assert(sizeof(DecodeKV8Smem<D, NT>) <= 113 * 1024, "two CTAs of an SM share its shared memory");
  cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  return hx_launch_pdl_cluster(k, dim3((unsigned)(a.clusters * kKV8CL)), dim3(kKV8Warps * 32), smem, st, kKV8CL, a);
}

cudaError_t attn_decode_kv8_launch(const AttnDecodeKV8Args& a, cudaStream_t st) {
  cudaError_t e = cudaSuccess;
  kv8_dispatch(a.c.D, a.c.fp8, [&](auto d, auto fp8) {
    constexpr int D = decltype(d)::value;
    constexpr bool F = decltype(fp8)::value;
    if (a.NT == 1) {
      e = launch_decode<D, 1, F>(a, st);
    } else if constexpr (D <= 128) {
      e = launch_decode<D, 2, F>(a, st);
    } else {
      e = cudaErrorInvalidValue;
    }
  });
  return e;
}

}  // namespace hx
