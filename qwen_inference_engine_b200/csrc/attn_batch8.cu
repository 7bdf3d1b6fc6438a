// attn_batch8.cu -- attention of a step's rows over a cache in 8 bits (kv8.cuh): requests with any number of rows, causal behind their cached positions, with an optional window
// (qie_attention_batch8).
//
//   out_t = sum_j 2^(x_tj - m) 2^ev_j v_j / sum_j 2^(x_tj - m),  x_tj = s 2^ek_j (q_t . k_j) over the positions j that row t sees, m their running maximum, k_j and v_j codes
//
// Codes become fp16 exactly.  A row's query is brought to fp16 by a power of two of its own, which loses nothing either, so scores are those of the values that the cache stands for,
// summed in fp32.  Weights are fp16 in the product with the values (2^-11 of themselves; 2^12 times themselves and times their value's scale, so that none of at least 2^-26 of the
// largest gets fewer bits), their sums fp32.
//
// An item is a kv head of a request and a block of its tokens, its rows (token, query head of the group); items are shared out over the CTAs as in attn_batch.cu.
#include <cuda.h>

#include <algorithm>

#include "attn_batch_split.cuh"
#include "common.cuh"
#include "kernels.h"
#include "kv8.cuh"
#include "launch.h"
#include "tc_ptx.cuh"

namespace qie {
namespace {

constexpr float LAG = 3.f;  // weights are at most 2^LAG: with 2^12 below the largest fp16
constexpr int P_EXP = 12;

// ---------------------------------------------------------------- blocks of at most 16 rows
constexpr int ROWS_F = 16, THR_F = 256, WARPS_F = THR_F / 32;

// (volatile: instructions that a whole warp executes together stay where they are, between what brings its threads together)
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_h(float a, float b) {  // a in the low half
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %2, %1;" : "=r"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void ld_shared_v4(uint32_t at, uint32_t (&r)[4]) {
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
// the power of two that brings a row whose largest element has these bits to fp16, and back (an infinity or no number: no number)
__device__ __forceinline__ void query_scale(uint32_t amax, float& there, float& back) {
  const uint32_t e = max(amax >> 23, 14u);
  there = __uint_as_float((267u - e) << 23), back = __uint_as_float((e - 13u) << 23);
  if (e >= 255) there = back = __uint_as_float(0x7fc00000u);
}

// keys and values on their way to a warp: units of 16 keys
template <int HD>
struct Ring {
  static constexpr int UNIT = 16 * HD, STAGES = HD == 128 ? 3 : 4, WARP = STAGES * 2 * UNIT;
};
template <int HD>
constexpr int SMEM_F = WARPS_F * Ring<HD>::WARP;

// A warp takes every eighth unit of 16 keys of the CTA's stretch, by copies into a ring of its own: keys from there as the rows of a product K Q^T, the weights by a transposition of
// 8 x 8 into fragments of V^T P^T, values with neighbouring keys' bytes beside each other.  The columns of a row are numbered so that a lane's are 16 bytes together.  No barrier but the
// warp's own; the warps' results are added up at the end of a piece.
template <int HD, int CODE, int NB>
__global__ void __launch_bounds__(THR_F, NB == 1 ? 2 : 1) attn_few8_kernel(BatchAttnArgs a, Kv8Geom kv, JoinShape sh, int tt) {
  constexpr int C = HD / 64, VW = HD / 32, MB = HD / 16;  // 16-byte pieces of a key row a lane; words of a value row a lane; blocks of 16 columns
  constexpr int UNIT = Ring<HD>::UNIT, ST = Ring<HD>::STAGES;
  static_assert(NB * 8 * HD * 4 <= Ring<HD>::WARP, "a warp's results take its ring's place");
  extern __shared__ __align__(128) unsigned char s_ring[];  // [warp][stage][k|v][key][column], and in its place the warp's results [row][column]
  __shared__ long long s_sums[THR_F / 32];
  __shared__ Walk s_walk;
  __shared__ float s_m[WARPS_F][NB * 8], s_l[WARPS_F][NB * 8];
  __shared__ int s_r[WARPS_F];
  __shared__ uint8_t s_scale[WARPS_F][ST][32];
  float* s_o = reinterpret_cast<float*>(s_ring);
  pdl_wait();
  pdl_trigger();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const uint32_t ring = smem_u32(s_ring) + warp * Ring<HD>::WARP;
  // 16-byte pieces of a row lie in an order of the row's, so that what lanes read together is in different banks
  auto k_at = [](int row, int piece) { return HD == 128 ? row * 128 + ((piece ^ ((row & 1) << 2)) << 4) : row * 64 + (piece << 4); };
  auto v_at = [](int row, int piece) { return HD == 128 ? row * 128 + ((piece ^ (row & 6)) << 4) : row * 64 + ((piece ^ ((row >> 1) & 3)) << 4); };
  if (tid == 0) s_walk.left = 0;
  const auto [share, x1] = find_stretch<THR_F>(a, tt, s_sums, &s_walk);
  __syncthreads();
  Walk walk = s_walk;
  JoinInfo* info = reinterpret_cast<JoinInfo*>(a.work);
  float* parts = reinterpret_cast<float*>(info + gridDim.x);
  if (tid == 0) info[blockIdx.x].parts = 0;
  Piece p;
  while (walk.next(a, tt, p)) {
    const int sub = p.kvh % sh.subs, kvh = p.kvh / sh.subs, G = min(sh.g, sh.group - sub * sh.g), rows = p.tokens * G;
    const size_t head0 = (size_t)kvh * sh.group + sub * sh.g;
    const int low0 = a.window > 0 ? max(0, p.pos0 - a.window + 1) : 0, low1 = a.window > 0 ? max(0, p.pos0 + p.tokens - a.window) : 0;  // of the first and the last token
    const int end = p.pos0 + p.tokens, k_lo = max(p.key0 + p.begin * AB_TK, low0 & ~15), k_hi = min(p.key0 + p.end * AB_TK, end);
    const int units = (k_hi - k_lo + 15) / 16;
    const int* bt = a.block_table + (size_t)p.slot * a.max_pages;
    const int P = kv.page_size, v_off = kv.n_kv * P;
    // the key of the unit that is the lane's (lanes 16 .. 31 the same again): its vector in the pool
    auto vec_of = [&](int u) {
      const int key = min(k_lo + u * 16 + (lane & 15), k_hi - 1), pg = key / P;
      int page = bt[pg];
      if (page < 0 || page >= kv.n_pages) page = 0;
      return ((page * kv.n_layers + a.layer) * 2 * kv.n_kv + kvh) * P + (key - pg * P);
    };
    auto copy = [&](int vec, int stage) {
      constexpr int PIECES = HD / 16, EACH = 16 * PIECES / 32;
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
        const int row = (i * 32 + lane) / PIECES, piece = lane % PIECES;
        const int r = __shfl_sync(0xffffffffu, vec, row);
        const uint8_t* src = kv.codes + (size_t)r * HD + piece * 16;
        cp_async16(ring + stage * 2 * UNIT + k_at(row, piece), src);
        cp_async16(ring + stage * 2 * UNIT + UNIT + v_at(row, piece), src + (size_t)v_off * HD);
      }
    };
    auto scale_of = [&](int vec) { return kv.scale[vec + (lane >> 4) * v_off]; };  // lanes 0 .. 15: keys', 16 .. 31: values'
    // ---- the first units on their way, and the vectors of the one behind them
    uint8_t first[ST - 1], pend = 0;
    int vec_next = 0, pend_at = -1;
#pragma unroll
    for (int s = 0; s < ST - 1; ++s) {
      const int u = warp + s * WARPS_F;
      if (u < units) {
        const int vec = vec_of(u);
        copy(vec, s);
        first[s] = scale_of(vec);
      }
      cp_async_commit();
    }
    if (warp + (ST - 1) * WARPS_F < units) vec_next = vec_of(warp + (ST - 1) * WARPS_F);
    // ---- queries: the lane's columns of row g (and 8 + g)
    uint32_t q[NB][C][4][2];
    float qf[NB][2];
    int pos[NB][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int n = nb * 8 + g, tok = n / G;
      uint4 x[C][2];
#pragma unroll
      for (int c = 0; c < C; ++c) {
        x[c][0] = x[c][1] = make_uint4(0, 0, 0, 0);
        if (n < rows) {
          const uint4* src = reinterpret_cast<const uint4*>(a.q + (size_t)(p.t0 + tok) * a.q_stride + (head0 + n - tok * G) * HD + c * 64 + t * 16);
          x[c][0] = src[0], x[c][1] = src[1];
        }
      }
      uint32_t most = 0;
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t w[4] = {x[c][h].x, x[c][h].y, x[c][h].z, x[c][h].w};
#pragma unroll
          for (int j = 0; j < 4; ++j) most = max(most, max(w[j] << 16 & 0x7fff0000u, w[j] & 0x7fff0000u));
        }
      most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
      float there, back;
      query_scale(most, there, back);
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t w[4] = {x[c][h].x, x[c][h].y, x[c][h].z, x[c][h].w};
#pragma unroll
          for (int j = 0; j < 4; ++j) q[nb][c][2 * h + j / 2][j & 1] = pack_h(lo2f(w[j]) * there, hi2f(w[j]) * there);
        }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        qf[nb][e] = __shfl_sync(0xffffffffu, back, (2 * t + e) * 4) * a.scale_log2;
        pos[nb][e] = p.pos0 + min((nb * 8 + 2 * t + e) / G, p.tokens - 1);
      }
    }
    float o[NB][MB][4] = {}, m[NB][2], l[NB][2];
    int lr = 1;  // the largest scale of a value so far, as its byte
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) m[nb][0] = m[nb][1] = -INFINITY, l[nb][0] = l[nb][1] = 0.f;
#pragma unroll
    for (int s = 0; s < ST - 1; ++s)
      if (warp + s * WARPS_F < units) s_scale[warp][s][lane] = first[s];
    int stage = 0, into = ST - 1;  // of the unit at hand, and of the one that is asked for
    for (int u = warp; u < units; u += WARPS_F) {
      if (pend_at >= 0) s_scale[warp][pend_at][lane] = pend;  // (a step later than asked for)
      cp_async_wait<ST - 2>();
      __syncwarp();  // the unit is there, and nobody reads the one before any more
      pend_at = -1;
      if (u + (ST - 1) * WARPS_F < units) {
        copy(vec_next, into);
        pend = scale_of(vec_next), pend_at = into;
        if (u + ST * WARPS_F < units) vec_next = vec_of(u + ST * WARPS_F);
      }
      cp_async_commit();
      const int key0 = k_lo + u * 16;
      const bool edge = key0 + 16 > p.pos0 + 1 || key0 < low1;  // some row does not see some key of the unit
      const uint32_t at = ring + stage * 2 * UNIT;
      const uint8_t* sc = s_scale[warp][stage];
      // ---- scores: rows keys g and g + 8, columns rows 2t and 2t + 1
      float x[NB][4] = {};
#pragma unroll
      for (int c = 0; c < C; ++c) {
        uint32_t k0[4], k1[4];
        ld_shared_v4(at + k_at(g, c * 4 + t), k0);
        ld_shared_v4(at + k_at(g + 8, c * 4 + t), k1);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          uint32_t a0, a1, a2, a3;
          kv8_unpack<CODE>(k0[w], a0, a2);
          kv8_unpack<CODE>(k1[w], a1, a3);
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) mma_f16(x[nb], a0, a1, a2, a3, q[nb][c][w][0], q[nb][c][w][1]);
        }
      }
      uint32_t vr[4][VW];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = 2 * t + (i & 1) + 8 * (i >> 1);
        if constexpr (HD == 128) ld_shared_v4(at + UNIT + v_at(row, g), vr[i]);
        else asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(vr[i][0]), "=r"(vr[i][1]) : "r"(at + UNIT + v_at(row, g >> 1) + (g & 1) * 8) : "memory");
      }
      const uint32_t kb0 = sc[g], kb1 = sc[g + 8], vb0 = sc[g + 16], vb1 = sc[g + 24];
      const int top = (int)__reduce_max_sync(0xffffffffu, lane < 16 || sc[lane] == 255 ? 0u : (uint32_t)sc[lane]);
      float ks[2] = {kv8_scale(vb0 == 255 ? 255u : kb0), kv8_scale(vb1 == 255 ? 255u : kb1)};
      if (edge && CODE == KV8_E4M3) {  // values that are no numbers must not meet a zero weight: they are zero, and their keys' scores no numbers
        uint32_t bad = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t any = 0;
#pragma unroll
          for (int w = 0; w < VW; ++w) any |= kv8_nans(vr[i][w]);
          if (any) {
            bad |= 1u << (2 * t + (i & 1) + 8 * (i >> 1));
#pragma unroll
            for (int w = 0; w < VW; ++w) vr[i][w] = 0;
          }
        }
        bad = __reduce_or_sync(0xffffffffu, bad);
        if (bad) {
          // (the other lanes' columns of the key stay as they are: a row that sees it is no number by its score)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (bad >> (g + 8 * i) & 1) ks[i] = __uint_as_float(0x7fc00000u);
        }
      }
      if (top > lr) {  // the values' products so far, beside the new largest scale
        const float f = top - lr < 127 ? __uint_as_float((uint32_t)(127 - (top - lr)) << 23) : 0.f;
        lr = top;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int b = 0; b < MB; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[nb][b][e] *= f;
      }
      float pv[2];  // 2^12 times a value's scale beside the largest
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int e = max(1, (int)(i ? vb1 : vb0)) - lr + 127 + P_EXP;
        pv[i] = e > 0 && e < 255 ? __uint_as_float((uint32_t)e << 23) : 0.f;
      }
      bool grow = false;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[nb][e] *= ks[e >> 1] * qf[nb][e & 1];
          if (edge) {
            const int key = key0 + g + 8 * (e >> 1), at = pos[nb][e & 1];
            if (key > at || (a.window > 0 && key <= at - a.window)) x[nb][e] = -INFINITY;
          }
          grow |= x[nb][e] > m[nb][e & 1] + LAG;
        }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float mx = fmaxf(x[nb][e], x[nb][e + 2]);
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
            const float to = fmaxf(m[nb][e], mx), f = m[nb][e] > -INFINITY ? ex2_tc(m[nb][e] - to) : 1.f;
            m[nb][e] = to;
            l[nb][e] *= f;
#pragma unroll
            for (int b = 0; b < MB; ++b) o[nb][b][e] *= f, o[nb][b][e + 2] *= f;
          }
      }
      uint32_t pt[NB][2];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const float m0 = m[nb][0] > -INFINITY ? m[nb][0] : 0.f, m1 = m[nb][1] > -INFINITY ? m[nb][1] : 0.f;
        const float w0 = ex2_tc(x[nb][0] - m0), w1 = ex2_tc(x[nb][1] - m1), w2 = ex2_tc(x[nb][2] - m0), w3 = ex2_tc(x[nb][3] - m1);
        l[nb][0] += w0 + w2, l[nb][1] += w1 + w3;
        pt[nb][0] = transpose_8x8(pack_h(w0 * pv[0], w1 * pv[0]));
        pt[nb][1] = transpose_8x8(pack_h(w2 * pv[1], w3 * pv[1]));
      }
#pragma unroll
      for (int w = 0; w < VW; ++w) {
        uint32_t f[2][4];  // columns 4w .. 4w + 3 of two keys each
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          kv8_unpack<CODE>(__byte_perm(vr[2 * h][w], vr[2 * h + 1][w], 0x5140), f[h][0], f[h][1]);
          kv8_unpack<CODE>(__byte_perm(vr[2 * h][w], vr[2 * h + 1][w], 0x7362), f[h][2], f[h][3]);
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          mma_f16(o[nb][2 * w], f[0][0], f[0][1], f[1][0], f[1][1], pt[nb][0], pt[nb][1]);
          mma_f16(o[nb][2 * w + 1], f[0][2], f[0][3], f[1][2], f[1][3], pt[nb][0], pt[nb][1]);
        }
      }
      if (++stage == ST) stage = 0;
      if (++into == ST) into = 0;
    }
    cp_async_wait<0>();
    __syncwarp();
    // ---- the warps' results together
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[nb][e] += __shfl_xor_sync(0xffffffffu, l[nb][e], d);
        const int n = nb * 8 + 2 * t + e;
        if (g == 0) s_m[warp][n] = m[nb][e], s_l[warp][n] = l[nb][e];
        float* dst = s_o + warp * (Ring<HD>::WARP / 4) + n * HD + g * (HD / 8);
#pragma unroll
        for (int b = 0; b < MB; ++b) *reinterpret_cast<float2*>(dst + 2 * b) = make_float2(o[nb][b][e], o[nb][b][e + 2]);
      }
    if (lane == 0) s_r[warp] = lr;
    __syncthreads();
    const bool whole = p.whole();
    for (int i = tid; i < rows * (HD / 4); i += THR_F) {
      const int n = i / (HD / 4), c = i - n * (HD / 4);
      float top = -INFINITY, sum = 0.f;
      int r = 1;
#pragma unroll
      for (int w = 0; w < WARPS_F; ++w) top = fmaxf(top, s_m[w][n]), r = max(r, s_r[w]);
      float4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < WARPS_F; ++w) {
        const float f = weight(s_m[w][n], s_l[w][n], top);
        sum += s_l[w][n] * f;
        const float fo = f * (r - s_r[w] < 127 ? __uint_as_float((uint32_t)(127 - (r - s_r[w])) << 23) : 0.f);
        const float4 x = *reinterpret_cast<const float4*>(s_o + w * (Ring<HD>::WARP / 4) + n * HD + c * 4);
        if (fo != 0.f) acc.x += x.x * fo, acc.y += x.y * fo, acc.z += x.z * fo, acc.w += x.w * fo;
      }
      const float back = __uint_as_float((uint32_t)r << 23) * (1.f / (1 << P_EXP));
      if (whole) {
        const float f = sum > 0.f ? back / sum : sum;
        const int tok = n / G;
        *reinterpret_cast<uint2*>(a.out + (size_t)(p.t0 + tok) * a.out_stride + (head0 + n - tok * G) * HD + c * 4) =
            make_uint2(pack2f(acc.x * f, acc.y * f), pack2f(acc.z * f, acc.w * f));
      } else {
        float* part = parts + ((size_t)blockIdx.x * 2 + (p.begin == 0)) * PART<HD, ROWS_F>;
        if (c == 0) part[ROWS_F * HD + n] = top, part[ROWS_F * HD + ROWS_F + n] = sum;
        *reinterpret_cast<float4*>(part + (c * ROWS_F + n) * 4) = make_float4(acc.x * back, acc.y * back, acc.z * back, acc.w * back);
      }
    }
    if (tid == 0 && !whole && p.begin == 0) info[blockIdx.x] = JoinInfo{p.t0, p.tokens, p.kvh, (int)quotient(x1 - p.left + p.tiles - 1, share) - (int)blockIdx.x + 1};
    __syncthreads();
  }
}

template <int HD, int CODE, int NB>
cudaError_t launch_few(const BatchAttnArgs& a, const Kv8Geom& kv, const JoinShape& sh, int tt, cudaStream_t st) {
  static PerDeviceOnce set;
  if (set.need()) {
    const cudaError_t e = cudaFuncSetAttribute(attn_few8_kernel<HD, CODE, NB>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_F<HD>);
    if (e != cudaSuccess) return e;
    set.done();
  }
  const int ctas = 2 * a.num_sms;
  BatchAttnArgs b = a;
  b.kv.n_kv *= sh.subs;
  const cudaError_t e = launched(launch_k(attn_few8_kernel<HD, CODE, NB>, dim3(ctas), dim3(THR_F), SMEM_F<HD>, st, b, kv, sh, tt));
  return e != cudaSuccess ? e : launch_join<HD, ROWS_F>(a, sh, ctas, st);
}

}  // namespace

size_t attention_batch8_work(int hd, int num_sms) { return (size_t)2 * num_sms * (sizeof(JoinInfo) + 2 * (hd == 64 ? PART<64, ROWS_F> : PART<128, ROWS_F>) * sizeof(float)); }

cudaError_t launch_attention_batch8(const BatchAttnArgs& a, const Kv8Geom& kv, cudaStream_t st) {
  const int group = a.n_q / kv.n_kv, g = std::min(group, ROWS_F), tt = ROWS_F / g;
  const JoinShape sh{g, group, (group + g - 1) / g};
  const bool one = group <= 8 && a.n_tok <= a.n_req;  // (a row a request: eight rows are enough)
  auto go = [&](auto hd, auto code) {
    constexpr int HD = decltype(hd)::value, CODE = decltype(code)::value;
    return one ? launch_few<HD, CODE, 1>(a, kv, sh, 8 / g, st) : launch_few<HD, CODE, 2>(a, kv, sh, tt, st);
  };
  using std::integral_constant;
  if (kv.hd == 64) return kv.code == KV8_E4M3 ? go(integral_constant<int, 64>(), integral_constant<int, KV8_E4M3>()) : go(integral_constant<int, 64>(), integral_constant<int, KV8_INT8>());
  return kv.code == KV8_E4M3 ? go(integral_constant<int, 128>(), integral_constant<int, KV8_E4M3>()) : go(integral_constant<int, 128>(), integral_constant<int, KV8_INT8>());
}

}  // namespace qie
