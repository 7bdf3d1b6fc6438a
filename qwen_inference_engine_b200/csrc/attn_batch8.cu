// attn_batch8.cu -- attention of a step's rows over a cache in 8 bits (kv8.cuh): requests with any number of rows, causal behind their cached positions, with an optional window
// (qie_attention_batch8).
//
//   out_t = sum_j 2^(x_tj - m) 2^ev_j v_j / sum_j 2^(x_tj - m),  x_tj = s 2^ek_j (q_t . k_j) over the positions j that row t sees, m their running maximum, k_j and v_j codes
//
// Codes become fp16 exactly, in larger blocks with a power of two beside them that a tile's keys, or values, have in common.  A row's query is brought to fp16 by a power of two of its own, which
// loses nothing down to 2^-31 of its largest element, and scores are summed in fp32.  A row goes by what it sees and by nothing beside it: m is its own running maximum, and its weights, which are fp16 in the product with the values
// (2^-11 of themselves), stand there times their values' scales beside the largest such product that the row itself has met (a reference of their own), so that none is off by more than 2^-31 of that,
// in larger blocks 2^-23, where a tile has one scale for values that are at most 2^8 apart.  Weights' sums are fp32.
//
// An item is a kv head of a request and a block of its tokens, its rows (token, query head of the group); items are shared out over the CTAs as in attn_batch.cu.  There are two kernels: for blocks
// of at most 16 rows (decode), which memory bounds, one that keeps a unit of keys and values in registers between loads and products, and for larger blocks one on tcgen05 / TMEM.
//
// What bounds them (B200, in a graph; the cache as it is read, with its scales).
//   Few rows.  64 at 1434 positions on average, 28 heads of 128 on 4, e4m3, 96 MB: 30.2 us (over a bf16 cache 42.8).  2.3 us pass before the first copies (the requests' numbers, the search for a
//   CTA's stretch), then units come at 4.9 TB/s until the median CTA ends at 21 us and the last one at 25, and the kernel that joins takes the rest.  4 at 70000 positions, 12 heads on 2, int8,
//   144 MB: 38.3 (62.3).  One at 700, 14 heads of 64 on 2: 9.1 (9.4), the plan, one tile's latency and the join.
//   Larger blocks.  8192 rows of 28 heads of 128 on 4: e4m3 563 us, 855 TFLOP/s, int8 573 (over a bf16 cache 491, which has nothing to convert).  A tile of 64 keys of 256 rows has 1024 cycles
//   of exponentials, 1280 of products and 1500 of shared memory's bandwidth (its products' operands, codes and fp16 in and out) and takes 2600.  At 586 us it was 6 % less without the exponentials'
//   instructions, 13 % without the conversion's arithmetic, 6 % without maxima, 11 % with an eighth of Q K^T: several chains of a tile (scores, softmax, product; copy, conversion) are about as
//   long as each other, and their code only just has room in the instruction caches: forms of the same instructions in other places took from 547 to 890 us.  An item's beginning and end, at
//   which both row tiles drain, cost 7 us.  A tile that is gone through twice takes twice as long: one key or value of each 64 2^20 below the others 1041 us, all values of 2^0 .. 2^60 4614.
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

// The weights' reference follows a row's maximum where it has fallen behind by more than 2^8: weights by 2^7 are at most 2^15 then, below the largest fp16.
constexpr int LAG_EXP = 8, P_EXP = 7;
constexpr float LAG = LAG_EXP;
constexpr float NOTHING = -3.4e38f;  // the reference of a row that has seen nothing: below every score, and a number
// from sums beside the reference of products, 2^rel times the one of weights (2^P_EXP times themselves), to sums beside that one, but for 2^LAG_EXP: weights' sums are at most so much more than
// they would be beside their maximum, and the factor must not leave the range ahead of them.  A row that has seen no value but zeros: 0
__device__ __forceinline__ float result_scale(float rel) { return rel > -INFINITY ? ex2_tc(rel - (float)(P_EXP + LAG_EXP)) : 0.f; }
// a 16-byte piece of a row in shared memory: in the order that TMA gives with a swizzle over a row's bytes
template <int HD>
__device__ __forceinline__ int piece_at(int row, int piece) {
  return row * HD + ((HD == 128 ? piece ^ (row & 7) : piece ^ (row >> 1 & 3)) << 4);
}

// ---------------------------------------------------------------- blocks of at most 16 rows
constexpr int ROWS_F = 16;

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

// keys and values on their way to a warp, in units of 32 keys; two CTAs an SM
template <int HD>
struct Ring {
  static constexpr int WARPS = HD == 128 ? 6 : 8, THR = WARPS * 32;
  static constexpr int UNIT = 32 * HD, STAGES = HD == 128 ? 2 : 3, WARP = STAGES * 2 * UNIT, SMEM = WARPS * WARP + 1024;
};

// A warp takes units of 32 keys of the CTA's stretch, one of WARPS, by copies into a ring of its own (TMA boxes of as many rows as divide a page, or for pages of other than multiples of
// four positions 16 bytes a lane): keys from there as the rows of a product K Q^T, the weights by a transposition of 8 x 8 into fragments of V^T P^T, values with neighbouring keys' bytes
// beside each other.  The columns of a row are numbered so that a lane's are 16 bytes together.  No barrier but the warp's own; the warps' results are added up at the end of a piece.
template <int HD, int CODE, int NB, bool TMA>
__global__ void __launch_bounds__(Ring<HD>::THR, NB == 1 ? 2 : 1) attn_few8_kernel(BatchAttnArgs a, Kv8Geom kv, JoinShape sh, int tt, int box, const __grid_constant__ CUtensorMap cm) {
  constexpr int C = HD / 64, VW = HD / 32, MB = HD / 16;  // 16-byte pieces of a key row a lane; words of a value row a lane; blocks of 16 columns
  constexpr int UNIT = Ring<HD>::UNIT, ST = Ring<HD>::STAGES, WARPS_F = Ring<HD>::WARPS, THR_F = Ring<HD>::THR;
  static_assert(NB * 8 * HD * 4 <= Ring<HD>::WARP, "a warp's results take its ring's place");
  extern __shared__ __align__(1024) unsigned char smem_raw[];  // [warp][stage][k|v][key][column], and in its place the warp's results [row][column]
  __shared__ long long s_sums[THR_F / 32];
  __shared__ Walk s_walk;
  __shared__ float s_m[WARPS_F][NB * 8], s_l[WARPS_F][NB * 8], s_rel[WARPS_F][NB * 8];
  __shared__ uint8_t s_scale[WARPS_F][ST][64];  // keys', values'
  __shared__ unsigned long long s_bar[WARPS_F][ST];
  __shared__ int dead_s;
  volatile int* dead = &dead_s;
  unsigned char* s_ring = smem_raw + ((smem_u32(smem_raw) + 1023u & ~1023u) - smem_u32(smem_raw));
  float* s_o = reinterpret_cast<float*>(s_ring);
  if (TMA && threadIdx.x == 32) asm volatile("prefetch.tensormap [%0];" ::"l"(&cm) : "memory");
  pdl_wait();  // (behind the kernel of larger blocks too, with which it shares nothing: what that one waited for is there for this one's loads behind a wait of its own)
  pdl_trigger();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const uint32_t ring = smem_u32(s_ring) + warp * Ring<HD>::WARP;
  if (TMA && lane == 0) {
    for (int i = 0; i < ST; ++i) mbar_init_tc(smem_u32(&s_bar[warp][i]), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (tid == 0) dead_s = 0;
  if (tid == 0) s_walk.left = 0;
  const auto [share, x1] = find_stretch<THR_F>(a, tt, s_sums, &s_walk);
  __syncthreads();
  Walk walk = s_walk;
  JoinInfo* info = reinterpret_cast<JoinInfo*>(a.work);
  float* parts = reinterpret_cast<float*>(info + gridDim.x);
  if (tid == 0) info[blockIdx.x].parts = 0;
  Piece p;
  int J = 0;  // (TMA) units that the warp had in the pieces before
  while (walk.next(a, tt, p)) {
    const int sub = p.kvh % sh.subs, kvh = p.kvh / sh.subs, G = min(sh.g, sh.group - sub * sh.g), rows = p.tokens * G;
    const size_t head0 = (size_t)kvh * sh.group + sub * sh.g;
    const int low0 = a.window > 0 ? max(0, p.pos0 - a.window + 1) : 0, low1 = a.window > 0 ? max(0, p.pos0 + p.tokens - a.window) : 0;  // of the first and the last token
    const int end = p.pos0 + p.tokens, k_lo = max(p.key0 + p.begin * AB_TK, low0 & ~31), k_hi = min(p.key0 + p.end * AB_TK, end);
    const int units = (k_hi - k_lo + 31) / 32, n = units > warp ? (units - warp + WARPS_F - 1) / WARPS_F : 0;  // the piece's, the warp's
    const int* bt = a.block_table + (size_t)p.slot * a.max_pages;
    const int P = kv.page_size, v_off = kv.n_kv * P;
    auto vec_of = [&](int j) {  // of the lane's key of unit j: its vector in the pool
      const int key = min(k_lo + (warp + j * WARPS_F) * 32 + lane, k_hi - 1), pg = key / P;
      int page = bt[pg];
      if (page < 0 || page >= kv.n_pages) page = 0;
      return ((page * kv.n_layers + a.layer) * 2 * kv.n_kv + kvh) * P + (key - pg * P);
    };
    auto copy = [&](int vec, int stage) {
      const uint32_t dst = ring + stage * 2 * UNIT;
      if constexpr (TMA) {
        const uint32_t bar = smem_u32(&s_bar[warp][stage]);
        if (lane == 0) asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"((uint32_t)(2 * UNIT)) : "memory");
        __syncwarp();
        if ((lane & (box - 1)) == 0) {  // (keys behind the last one: rows of the pool, or zeros behind it)
          asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst + lane * HD), "l"(&cm), "r"(bar), "r"(0), "r"(vec) : "memory");
          asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst + UNIT + lane * HD), "l"(&cm), "r"(bar), "r"(0), "r"(vec + v_off) : "memory");
        }
        __syncwarp();
      } else {
        constexpr int PIECES = HD / 16;
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
          const int row = (i * 32 + lane) / PIECES, piece = lane % PIECES, r = __shfl_sync(0xffffffffu, vec, row);
          const uint8_t* src = kv.codes + (size_t)r * HD + piece * 16;
          cp_async16(dst + piece_at<HD>(row, piece), src);
          cp_async16(dst + UNIT + piece_at<HD>(row, piece), src + (size_t)v_off * HD);
        }
        cp_async_commit();
      }
    };
    // ---- the first units on their way, and the vectors of the one behind them
    uint8_t sk[ST - 1], sv[ST - 1];
    int next = 0, pend_at = -1;
#pragma unroll
    for (int s = 0; s < ST - 1; ++s)
      if (s < n) {
        const int vec = vec_of(s);
        copy(vec, (J + s) % ST);
        sk[s] = kv.scale[vec], sv[s] = kv.scale[vec + v_off];
      } else if (!TMA) {
        cp_async_commit();
      }
    if (ST - 1 < n) next = vec_of(ST - 1);
    // ---- queries: the lane's columns of row g (and 8 + g)
    uint32_t q[NB][C][4][2];
    float qf[NB][2];
    int pos[NB][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int r = nb * 8 + g, tok = r / G;
      uint4 x[C][2];
#pragma unroll
      for (int c = 0; c < C; ++c) {
        x[c][0] = x[c][1] = make_uint4(0, 0, 0, 0);
        if (r < rows) {
          const uint4* src = reinterpret_cast<const uint4*>(a.q + (size_t)(p.t0 + tok) * a.q_stride + (head0 + r - tok * G) * HD + c * 64 + t * 16);
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
    // a row's references: m of its weights (l), and rel beside m of its weights times their values' scales (o); both are the row's own, of keys that it sees
    float o[NB][MB][4] = {}, m[NB][2], l[NB][2], rel[NB][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) m[nb][0] = m[nb][1] = rel[nb][0] = rel[nb][1] = NOTHING, l[nb][0] = l[nb][1] = 0.f;
#pragma unroll
    for (int s = 0; s < ST - 1; ++s)
      if (s < n) s_scale[warp][(J + s) % ST][lane] = sk[s], s_scale[warp][(J + s) % ST][32 + lane] = sv[s];
    int stage = J % ST;
    for (int j = 0; j < n; ++j) {
      if (pend_at >= 0) s_scale[warp][pend_at][lane] = sk[0], s_scale[warp][pend_at][32 + lane] = sv[0];  // (a step later than asked for)
      if constexpr (TMA) mbar_wait_short_tc(smem_u32(&s_bar[warp][stage]), (uint32_t)((J + j) / ST & 1), dead);
      else cp_async_wait<ST - 2>();
      __syncwarp();  // the unit is there, and nobody reads the one before any more
      pend_at = -1;
      if (j + ST - 1 < n) {
        pend_at = stage == 0 ? ST - 1 : stage - 1;
        copy(next, pend_at);
        sk[0] = kv.scale[next], sv[0] = kv.scale[next + v_off];
        if (j + ST < n) next = vec_of(j + ST);
      } else if (!TMA) {
        cp_async_commit();
      }
      const int key0 = k_lo + (warp + j * WARPS_F) * 32;
      const bool edge = key0 + 32 > p.pos0 + 1 || key0 < low1;  // some row does not see some key of the unit
      const uint32_t at = ring + stage * 2 * UNIT;
      const uint8_t* sc = s_scale[warp][stage];
      // ---- scores: rows keys g, g + 8, g + 16 and g + 24, columns rows 2t and 2t + 1; two sums each, of every other product (a chain of eight would be the unit's longest)
      float x[NB][2][4];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        float y[NB][2][4] = {};
#pragma unroll
        for (int c = 0; c < C; ++c) {
          uint32_t k0[4], k1[4];
          ld_shared_v4(at + piece_at<HD>(kb * 16 + g, c * 4 + t), k0);
          ld_shared_v4(at + piece_at<HD>(kb * 16 + g + 8, c * 4 + t), k1);
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            uint32_t a0, a1, a2, a3;
            kv8_unpack<CODE>(k0[w], a0, a2);
            kv8_unpack<CODE>(k1[w], a1, a3);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) mma_f16(y[nb][w & 1], a0, a1, a2, a3, q[nb][c][w][0], q[nb][c][w][1]);
          }
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int e = 0; e < 4; ++e) x[nb][kb][e] = y[nb][0][e] + y[nb][1][e];
      }
      uint32_t kb_[4], vb_[4];  // scales of the keys g + 8 i
#pragma unroll
      for (int i = 0; i < 4; ++i) kb_[i] = sc[g + 8 * i], vb_[i] = sc[32 + g + 8 * i];
      uint32_t bad = 0;
      if (edge && CODE == KV8_E4M3) {  // values that are no numbers must not meet a zero weight: they are zero, and their keys' scores no numbers
#pragma unroll 1
        for (int i = 0; i < HD / 16; ++i) {  // two keys a step; 16 or 8 bytes a lane
          const int row = i * (512 / HD) + lane / (HD / 16), piece = lane % (HD / 16);
          const uint32_t where = at + UNIT + piece_at<HD>(row, piece);
          uint32_t c[4];
          ld_shared_v4(where, c);
          if (kv8_nans(c[0]) | kv8_nans(c[1]) | kv8_nans(c[2]) | kv8_nans(c[3])) {
            bad |= 1u << row;
            asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(where), "r"(0u) : "memory");
          }
        }
        bad = __reduce_or_sync(0xffffffffu, bad);
        if (TMA) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // (a copy takes the place)
        __syncwarp();
      }
      float ve[4];  // the values' scales, as exponents (of zeros: minus infinity)
#pragma unroll
      for (int i = 0; i < 4; ++i) ve[i] = vb_[i] == 0 ? -INFINITY : (float)((int)vb_[i] - 127);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float ks = kv8_scale(vb_[i] == 255 || (bad >> (g + 8 * i) & 1) ? 255u : kb_[i]);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float& y = x[nb][i >> 1][(i & 1) * 2 + e];
            y = __fmul_rn(y, ks * qf[nb][e]);  // (rounded here: its difference from the largest is that of rounded scores)
            if (edge) {
              const int key = key0 + g + 8 * i, pos_ = pos[nb][e];
              if (key > pos_ || (a.window > 0 && key <= pos_ - a.window)) y = -INFINITY;
            }
          }
      }
      // exponents of weights beside their reference, and for the product 2^7 times themselves and their values' scales, beside the reference of those
      float p[NB][2][4];
      bool grow = false;
      auto exponents = [&](int nb, int i, int e) {
        const int at = (i & 1) * 2 + e;
        const float d = x[nb][i >> 1][at] - m[nb][e];
        p[nb][i >> 1][at] = d + (ve[i] + (P_EXP - rel[nb][e]));
        return d;
      };
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float d = exponents(nb, i, e);
            grow |= d > LAG || p[nb][i >> 1][(i & 1) * 2 + e] > LAG + P_EXP;
          }
      if (__any_sync(0xffffffffu, grow)) {
        // the rows' new references, and what there is so far beside them
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float mx = fmaxf(fmaxf(x[nb][0][e], x[nb][0][e + 2]), fmaxf(x[nb][1][e], x[nb][1][e + 2]));
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
            const float to = fmaxf(m[nb][e], mx);
            float rx = fmaxf(fmaxf((x[nb][0][e] - to) + ve[0], (x[nb][0][e + 2] - to) + ve[1]), fmaxf((x[nb][1][e] - to) + ve[2], (x[nb][1][e + 2] - to) + ve[3]));
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) rx = fmaxf(rx, __shfl_xor_sync(0xffffffffu, rx, d));
            const float before = fmaxf(rel[nb][e] + (m[nb][e] - to), NOTHING), f = ex2_tc(before - fmaxf(before, rx));  // (a number, where all values so far are zeros too)
            l[nb][e] *= ex2_tc(m[nb][e] - to);
            m[nb][e] = to, rel[nb][e] = fmaxf(before, rx);
#pragma unroll
            for (int b = 0; b < MB; ++b) o[nb][b][e] *= f, o[nb][b][e + 2] *= f;
#pragma unroll
            for (int i = 0; i < 4; ++i) exponents(nb, i, e);
          }
      }
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        uint32_t vr[4][VW];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = kb * 16 + 2 * t + (i & 1) + 8 * (i >> 1);
          if constexpr (HD == 128) ld_shared_v4(at + UNIT + piece_at<HD>(row, g), vr[i]);
          else asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(vr[i][0]), "=r"(vr[i][1]) : "r"(at + UNIT + piece_at<HD>(row, g >> 1) + (g & 1) * 8) : "memory");
        }
        uint32_t pt[NB][2];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          l[nb][0] += ex2_tc(x[nb][kb][0] - m[nb][0]) + ex2_tc(x[nb][kb][2] - m[nb][0]), l[nb][1] += ex2_tc(x[nb][kb][1] - m[nb][1]) + ex2_tc(x[nb][kb][3] - m[nb][1]);
          pt[nb][0] = transpose_8x8(pack_h(ex2_tc(p[nb][kb][0]), ex2_tc(p[nb][kb][1])));
          pt[nb][1] = transpose_8x8(pack_h(ex2_tc(p[nb][kb][2]), ex2_tc(p[nb][kb][3])));
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
      }
      if (++stage == ST) stage = 0;
    }
    J += n;
    if (!TMA) cp_async_wait<0>();
    __syncwarp();
    // ---- the warps' results together
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[nb][e] += __shfl_xor_sync(0xffffffffu, l[nb][e], d);
        const int r = nb * 8 + 2 * t + e;
        if (g == 0) s_m[warp][r] = m[nb][e] > NOTHING ? m[nb][e] : -INFINITY, s_l[warp][r] = l[nb][e], s_rel[warp][r] = rel[nb][e];
        float* dst = s_o + warp * (Ring<HD>::WARP / 4) + r * HD + g * (HD / 8);
#pragma unroll
        for (int b = 0; b < MB; ++b) *reinterpret_cast<float2*>(dst + 2 * b) = make_float2(o[nb][b][e], o[nb][b][e + 2]);
      }
    __syncthreads();
    const bool whole = p.whole();
    for (int i = tid; i < rows * (HD / 4); i += THR_F) {
      const int n = i / (HD / 4), c = i - n * (HD / 4);  // a row, four columns
      float top = -INFINITY, sum = 0.f, r = -INFINITY;
#pragma unroll
      for (int w = 0; w < WARPS_F; ++w) top = fmaxf(top, s_m[w][n]);
      auto beside = [&](int w) { return s_m[w][n] > -INFINITY ? s_rel[w][n] + (s_m[w][n] - top) : -INFINITY; };  // the warp's reference of products, beside the row's maximum
#pragma unroll
      for (int w = 0; w < WARPS_F; ++w) r = fmaxf(r, beside(w));
      float4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < WARPS_F; ++w) {
        sum += s_l[w][n] * weight(s_m[w][n], s_l[w][n], top);
        const float at = beside(w), fo = at > -INFINITY ? ex2_tc(at - r) : 0.f;
        const float4 x = *reinterpret_cast<const float4*>(s_o + w * (Ring<HD>::WARP / 4) + n * HD + c * 4);
        if (fo != 0.f) acc.x += x.x * fo, acc.y += x.y * fo, acc.z += x.z * fo, acc.w += x.w * fo;
      }
      const float back = result_scale(r);
      if (whole) {
        const float f = *dead ? __int_as_float(0x7fc00000) : sum > 0.f ? back * ((1 << LAG_EXP) / sum) : sum;
        const int tok = n / G;
        *reinterpret_cast<uint2*>(a.out + (size_t)(p.t0 + tok) * a.out_stride + (head0 + n - tok * G) * HD + c * 4) =
            make_uint2(pack2f(acc.x * f, acc.y * f), pack2f(acc.z * f, acc.w * f));
      } else {
        float* part = parts + ((size_t)blockIdx.x * 2 + (p.begin == 0)) * PART<HD, ROWS_F>;
        const float all = back * (1 << LAG_EXP);
        if (c == 0) part[ROWS_F * HD + n] = top, part[ROWS_F * HD + ROWS_F + n] = *dead ? __int_as_float(0x7fc00000) : sum;
        *reinterpret_cast<float4*>(part + (c * ROWS_F + n) * 4) = make_float4(acc.x * all, acc.y * all, acc.z * all, acc.w * all);
      }
    }
    if (tid == 0 && !whole && p.begin == 0) info[blockIdx.x] = JoinInfo{p.t0, p.tokens, p.kvh, (int)quotient(x1 - p.left + p.tiles - 1, share) - (int)blockIdx.x + 1};
    if (TMA) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // (copies take the results' place)
    __syncthreads();
  }
  if (TMA && tid == 0) {
    drain_tc(dead);
    report_tc(dead, a.status);
  }
}

template <int HD, int CODE, int NB, bool TMA>
cudaError_t launch_few(const BatchAttnArgs& a, const Kv8Geom& kv, const JoinShape& sh, int tt, int box, bool behind, const TensorMap2D& cm, cudaStream_t st) {
  static PerDeviceOnce set;
  if (set.need()) {
    const cudaError_t e = cudaFuncSetAttribute(attn_few8_kernel<HD, CODE, NB, TMA>, cudaFuncAttributeMaxDynamicSharedMemorySize, Ring<HD>::SMEM);
    if (e != cudaSuccess) return e;
    set.done();
  }
  const int ctas = 2 * a.num_sms;
  BatchAttnArgs b = a;
  b.kv.n_kv *= sh.subs;
  b.rest = 7;  // (64 rows, heads of 128, with 3: CTAs with one piece end at 18 us, with two at 21)
  const cudaError_t e = launched(launch_k(attn_few8_kernel<HD, CODE, NB, TMA>, dim3(ctas), dim3(Ring<HD>::THR), Ring<HD>::SMEM, st, b, kv, sh, tt, box, *reinterpret_cast<const CUtensorMap*>(&cm)));
  return e != cudaSuccess || behind ? e : launch_join<HD, ROWS_F>(a, sh, ctas, st);
}

// ---------------------------------------------------------------- blocks of up to 256 rows
// On tcgen05 / TMEM, one CTA an SM.  Two tiles of 128 rows work on the same keys and values, so that a tile of 64 of those is brought to fp16 once for both; each is a chain of its own
// (scores, softmax, product), and while one is in its softmax the other one has the tensor pipe.
//   warps 0-3, 4-7 : the softmax of a row tile, a thread a row (= TMEM lane); queries into TMEM (the A operand of the scores, as the weights are of the products, so that shared memory
//                    feeds keys and values alone; with heads of 128 there is no room for both in TMEM, and they lie in shared memory), the rows of the result
//   warps 8-15     : codes to fp16 (keys, values): of a tile the powers of two beside its largest, which is a factor of all scores (keys) and of all weights (values), by the multiplication
//   warps 16, 17   : the products of a row tile
//   warp 18        : codes and scales by TMA, or, for pages of other than multiples of 16 positions, by 16-byte copies to the same places
//   warp 19        : of a tile the largest scales, which keys go by them, and every key's and value's factor
// Registers: 96 a thread at launch; 144, 64 and 64 behind the split, as many in all.
constexpr int ROWS_P = 256, THR_P = 20 * 32, TK = AB_TK;
constexpr int KBLK = TK * 128;  // [keys][64 columns] fp16 in 8-row swizzle atoms
constexpr int PLANS = 4, SLOTS = 16;  // tiles' factors; tiles' scales: warp 19 is at most PLANS tiles ahead of the conversion, and the softmax ST + 3 behind that
// A tile is brought to fp16 beside its largest scales, so keys far below those would lose bits and values would lie far from what the rows that see them go by.  Where keys' scales are more than
// KEYS_APART powers of two apart (a code's smallest step is fp16's smallest number then) or values' more than VALUES_APART, the tile is gone through again for those: scores, softmax and product
// of some of its keys at a time (TILE_PART), until all have been there (TILE_AGAIN: not yet).
// A word of a tile: its values' largest scale in the lowest byte, its keys' where a float has its exponent, and these.  TILE_CLEAR: some values are not for the product.
constexpr int TILE_AGAIN = 1 << 8, TILE_PART = 1 << 9, TILE_CLEAR = 1 << 10;
template <int CODE>
constexpr uint32_t KEYS_APART = CODE == KV8_E4M3 ? 15 : 24;
constexpr uint32_t VALUES_APART = 8;
constexpr uint32_t NONE_H2 = 0x7e007e00u, CLEAR_H2 = 0xffffffffu;  // factors: no numbers; (of values) zeros, whatever the codes
__device__ __forceinline__ bool far_below(uint32_t byte, uint32_t top, uint32_t apart) { return byte + apart < top; }  // (no numbers: above all)
// a key of zeros has its score beside any scale; a value of zeros is far below others, as its weight says nothing about their products
template <int CODE>
__device__ __forceinline__ bool key_far(uint32_t byte, uint32_t top) { return byte != 0 && far_below(byte, top, KEYS_APART<CODE>); }
template <int HD>
struct SmemP {
  static constexpr bool Q_TMEM = HD == 64;
  static constexpr int NB = HD / 64, RAW = HD == 64 ? 4 : 3, ST = 3;  // column blocks; stages of codes, and of keys and values
  static constexpr int CODES = TK * HD, TILE = NB * KBLK, QBLK = 128 * 128, QTILE = NB * QBLK;
  static constexpr int C = 0, K = RAW * 2 * CODES, V = K + ST * TILE, Q = V + ST * TILE, SC = Q + (Q_TMEM ? 0 : 2 * QTILE), BAR = SC + RAW * 2 * TK, TOTAL = BAR + 512 + 1024;
  static_assert(TOTAL <= 226 * 1024 && ST + PLANS + 3 <= SLOTS, "");
};
// D = F32, A = B = F16
__device__ __forceinline__ uint32_t idesc_h(int m, int n, bool b_mn) { return idesc_tc(m, n, b_mn) & ~((1u << 7) | (1u << 10)); }
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) { asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ uint32_t mul_h2(uint32_t a, uint32_t b) {
  asm("mul.rn.f16x2 %0, %0, %1;" : "+r"(a) : "r"(b));
  return a;
}
// 2^-d twice as fp16, d >= 0 (or, where nobody looks at what comes of it, any)
__device__ __forceinline__ uint32_t pow2_h2(int d) {
  const float f = __uint_as_float((uint32_t)max(127 - d, 0) << 23);
  return pack_h(f, f);
}

template <int HD, int CODE, bool TMA>
__global__ void __launch_bounds__(THR_P, 1) attn_prompt8_kernel(BatchAttnArgs a, Kv8Geom kv, int G, int tt, int out32, int box, const __grid_constant__ CUtensorMap cm) {
  using SM = SmemP<HD>;
  constexpr int ST = SM::ST, RAW = SM::RAW;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  __shared__ long long s_sums[THR_P / 32];
  __shared__ Walk s_walk, s_walks[THR_P / 32];
  __shared__ int dead_s;
  __shared__ int s_tile[2][SLOTS];               // of a row tile's tiles the words
  __shared__ unsigned long long s_in[2][SLOTS];  // TILE_PART: which keys
  __shared__ int s_plan[PLANS];                  // the words of the tiles that are to be brought to fp16, and of those each key's and value's factor, twice as fp16
  __shared__ uint32_t s_factor[PLANS][2][TK];
  volatile int* dead = &dead_s;
  if (TMA && threadIdx.x == 18 * 32) asm volatile("prefetch.tensormap [%0];" ::"l"(&cm) : "memory");
  const uint32_t s0 = (smem_u32(smem_raw) + 1023u) & ~1023u;
  unsigned char* smem = smem_raw + (s0 - smem_u32(smem_raw));
  // barriers: of a row tile queries, and by its tile's parity scores, weights and product; of the stages of codes, keys and values full and free; of the tiles' factors full and free
  const uint32_t bar_q = s0 + SM::BAR, bar_s = bar_q + 16, bar_p = bar_s + 32, bar_o = bar_p + 32, slot = bar_o + 32, raw_full = slot + 16, raw_free = raw_full + 8 * RAW, k_full = raw_free + 8 * RAW,
                 k_free = k_full + 8 * ST, v_full = k_free + 8 * ST, v_free = v_full + 8 * ST, plan_full = v_free + 8 * ST, plan_free = plan_full + 8 * PLANS;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    dead_s = 0, s_walk.left = 0;
    for (int i = 0; i < 2; ++i) mbar_init_tc(bar_q + 8 * i, 128);
    for (int i = 0; i < 4; ++i) mbar_init_tc(bar_s + 8 * i, 1), mbar_init_tc(bar_p + 8 * i, 128), mbar_init_tc(bar_o + 8 * i, 1);
    for (int i = 0; i < PLANS; ++i) mbar_init_tc(plan_full + 8 * i, 1), mbar_init_tc(plan_free + 8 * i, 8);
    for (int i = 0; i < RAW; ++i) mbar_init_tc(raw_full + 8 * i, TMA ? 1 : 64), mbar_init_tc(raw_free + 8 * i, 8);
    for (int i = 0; i < ST; ++i) mbar_init_tc(k_full + 8 * i, 4), mbar_init_tc(k_free + 8 * i, 2), mbar_init_tc(v_full + 8 * i, 4), mbar_init_tc(v_free + 8 * i, 2);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 16) {  // (ahead of the kernel before: 61440 of an SM's registers are this CTA's, so none of that kernel's that still wants TMEM columns is on the SM)
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  pdl_wait();
  pdl_trigger();
  const auto [share, x1] = find_stretch<THR_P>(a, tt, s_sums, &s_walk);
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  uint32_t tmem;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem) : "r"(slot));
  // TMEM: scores of 64 columns (the weights over them) of a row tile's two tiles at hand, its O, its queries
  auto t_s = [&](int g, int b) { return tmem + (uint32_t)((2 * g + b) * TK); };
  auto t_o = [&](int g) { return tmem + 4 * TK + (uint32_t)(g * HD); };
  auto t_q = [&](int g) { return tmem + 4 * TK + 2 * HD + (uint32_t)(g * (HD / 2)); };
  JoinInfo* info = reinterpret_cast<JoinInfo*>(a.work);
  float* parts = reinterpret_cast<float*>(info + gridDim.x);
  // the pieces of the stretch, every warp for itself; between them in shared memory (in registers they cost the softmax spills)
  if (lane == 0) s_walks[warp] = s_walk;
  __syncwarp();
  auto next_piece = [&](Piece& p) {
    Walk walk = s_walks[warp];
    const bool some = walk.next(a, tt, p);
    __syncwarp();
    if (lane == 0) s_walks[warp] = walk;
    __syncwarp();
    return some;
  };
  // the warp's tile again?  (Behind a wait that ran out words may be any; the warp goes on together.)
  auto once_more = [&](int word) { return __any_sync(0xffffffffu, word & TILE_AGAIN) && !__any_sync(0xffffffffu, *dead); };
  Piece p;
  int T = 0;  // tiles so far

  if (warp >= 16) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");  // (a warpgroup together)
    if (warp >= 18) {
      // ---- codes and scales
      const int P = kv.page_size, v_off = kv.n_kv * P;
      const int chunks = TMA ? TK / box : 1;  // of a tile
      uint8_t wait_sc[4];                     // (not TMA) the scales of the tile before
      int waits = -1;
      auto put_scales = [&]() {
        if (waits < 0) return;
#pragma unroll
        for (int j = 0; j < 4; ++j) smem[SM::SC + waits * 2 * TK + j * 32 + lane] = wait_sc[j];
        mbar_arrive_tc(raw_full + 8u * (uint32_t)waits);
      };
      while (warp == 18 && next_piece(p)) {
        const int* bt = a.block_table + (size_t)p.slot * a.max_pages;
        const int last_page = (p.limit - 1) / P, c0 = TMA ? p.key0 / box : 0;
        int held = c0 + p.begin * chunks, page_of = 0;  // a lane holds the page of chunk `held` + lane
        if (TMA) page_of = bt[min((held + lane) * box / P, last_page)];
        for (int i = p.begin; i < p.end; ++i, ++T) {
          const int st = T % RAW;
          if (T >= RAW) mbar_wait_short_tc(raw_free + 8u * st, (uint32_t)((T / RAW - 1) & 1), dead);
          __syncwarp();
          const uint32_t bar = raw_full + 8u * st, dst = s0 + SM::C + st * 2 * SM::CODES, sc = s0 + SM::SC + st * 2 * TK;
          if constexpr (TMA) {
            const int ch = c0 + i * chunks;
            if (ch + chunks > held + 32) {
              held = ch;
              page_of = bt[min((held + lane) * box / P, last_page)];
            }
            const int j = lane % 4;  // a chunk; lanes 0 .. 3 keys, 4 .. 7 values, 8 .. 15 their scales
            int page = __shfl_sync(0xffffffffu, page_of, (ch - held + j) & 31);
            if (page < 0 || page >= kv.n_pages) page = 0;
            const int at = min((ch + j) * box, last_page * P + P - box) % P;  // (chunks behind the last page repeat its end: their keys are masked)
            const int is_v = lane >> 2 & 1, row = ((page * kv.n_layers + a.layer) * 2 * kv.n_kv + p.kvh) * P + at + is_v * v_off;
            if (lane == 0) asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"((uint32_t)(2 * SM::CODES + 2 * TK)) : "memory");
            __syncwarp();
            if (j < chunks && lane < 8)
              asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                           ::"r"(dst + is_v * SM::CODES + j * box * HD), "l"(&cm), "r"(bar), "r"(0), "r"(row)
                           : "memory");
            if (j < chunks && lane >= 8 && lane < 16)
              asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                           ::"r"(sc + is_v * TK + j * box), "l"(kv.scale + row), "r"(box), "r"(bar)
                           : "memory");
            __syncwarp();
          } else {
            put_scales();
            // the lane's keys, lane and 32 + lane of the tile: their vectors
            int vec[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int key = min(p.key0 + i * TK + h * 32 + lane, p.limit - 1), pg = key / P;
              int page = bt[pg];
              if (page < 0 || page >= kv.n_pages) page = 0;
              vec[h] = ((page * kv.n_layers + a.layer) * 2 * kv.n_kv + p.kvh) * P + (key - pg * P);
              wait_sc[h] = kv.scale[vec[h]], wait_sc[2 + h] = kv.scale[vec[h] + v_off];
            }
            waits = st;
            constexpr int PIECES = HD / 16;
#pragma unroll
            for (int e = 0; e < TK * PIECES / 32; ++e) {
              const int row = (e * 32 + lane) / PIECES, piece = lane % PIECES;
              const int r = __shfl_sync(0xffffffffu, e * 32 / PIECES < 32 ? vec[0] : vec[1], row & 31);
              const uint8_t* src = kv.codes + (size_t)r * HD + piece * 16;
              const uint32_t to = dst + row * HD + ((HD == 128 ? piece ^ (row & 7) : piece ^ ((row >> 1) & 3)) << 4);
              cp_async16(to, src);
              cp_async16(to + SM::CODES, src + (size_t)v_off * HD);
            }
            cp_async_arrive(bar);
          }
        }
      }
      if (!TMA && warp == 18) put_scales();
      // ---- the tiles' largest scales and factors, of the lane's keys, lane and 32 + lane
      int T1 = 0, tiles = 0;  // tiles of the second row tile; tiles as they are copied
      while (warp == 19 && next_piece(p)) {
        const int low0 = a.window > 0 ? max(0, p.pos0 - a.window + 1) : 0, low1 = a.window > 0 ? max(0, p.pos0 + p.tokens - a.window) : 0, end = p.pos0 + p.tokens;
        const bool both = p.tokens * G > 128;  // (row tiles with rows)
        int R = p.begin;
#pragma unroll 1
        for (; R < p.end; ++R) {
          const int at = tiles + R - p.begin, rs = at % RAW, key = p.key0 + R * TK;
          const bool edge = key + TK > p.pos0 + 1 || key < low1;  // some row does not see some key of the tile
          mbar_wait_short_tc(raw_full + 8u * (uint32_t)rs, (uint32_t)((at / RAW) & 1), dead);
          __syncwarp();
          const unsigned char *vc = smem + SM::C + (rs * 2 + 1) * SM::CODES, *sc = smem + SM::SC + rs * 2 * TK;
          unsigned long long bad = 0;  // keys whose values are no numbers, where these must not meet a zero weight: zero values and scores that are no numbers
          if (edge && CODE == KV8_E4M3) {
#pragma unroll 1
            for (int e = 0; e < TK * HD / 512; ++e) {
              const uint4 c = *reinterpret_cast<const uint4*>(vc + (e * 32 + lane) * 16);
              if (kv8_nans(c.x) | kv8_nans(c.y) | kv8_nans(c.z) | kv8_nans(c.w)) bad |= 1ull << ((e * 32 + lane) * 16 / HD);
            }
            bad = __reduce_or_sync(0xffffffffu, (uint32_t)bad) | (unsigned long long)__reduce_or_sync(0xffffffffu, (uint32_t)(bad >> 32)) << 32;
          }
          uint32_t kb[2], vb[2];
          bool in[2];  // whether it is still to come
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int row = h * 32 + lane;
            kb[h] = sc[row], vb[h] = sc[TK + row], in[h] = !edge || (key + row >= low0 && key + row < end);
          }
          int word;
#pragma unroll 1
          do {
            uint32_t kt = 0, vt = 1;
            bool now[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              now[h] = in[h];
              if (in[h] && kb[h] != 255) kt = max(kt, kb[h]);
              if (in[h] && vb[h] != 255) vt = max(vt, vb[h]);
            }
            kt = __reduce_max_sync(0xffffffffu, kt), vt = __reduce_max_sync(0xffffffffu, vt);
            auto far = [&](int h) { return in[h] && (key_far<CODE>(kb[h], kt) || far_below(vb[h], vt, VALUES_APART)); };
            word = 0;
            if (__any_sync(0xffffffffu, far(0) || far(1))) {  // of the keys near the largest those whose values are near the largest of theirs; the others another time
              vt = 1;
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                now[h] = in[h] && !key_far<CODE>(kb[h], kt);
                if (now[h] && vb[h] != 255) vt = max(vt, vb[h]);
              }
              vt = __reduce_max_sync(0xffffffffu, vt);
#pragma unroll
              for (int h = 0; h < 2; ++h) now[h] = now[h] && !far_below(vb[h], vt, VALUES_APART);
              word = TILE_AGAIN;
            }
            const unsigned long long mask = __ballot_sync(0xffffffffu, now[0]) | (unsigned long long)__ballot_sync(0xffffffffu, now[1]) << 32;
            const bool none[2] = {vb[0] == 255 || (bad >> lane & 1), vb[1] == 255 || (bad >> 32 >> lane & 1)};
            if (edge || ~mask || __any_sync(0xffffffffu, none[0] || none[1])) word |= TILE_CLEAR;
            if (~mask) word |= TILE_PART;
            word |= (int)(kt << 23 | vt);
            const int pl = T % PLANS;
            if (T >= PLANS) mbar_wait_short_tc(plan_free + 8u * (uint32_t)pl, (uint32_t)((T / PLANS - 1) & 1), dead);
            __syncwarp();
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              s_factor[pl][0][h * 32 + lane] = none[h] || kb[h] == 255 ? NONE_H2 : kb[h] == 0 ? 0u : pow2_h2((int)(kt - kb[h]));
              s_factor[pl][1][h * 32 + lane] = none[h] || !now[h] ? CLEAR_H2 : vb[h] == 0 ? 0u : pow2_h2((int)(vt - vb[h]));
              in[h] = in[h] && !now[h];
            }
            if (lane == 0) {  // (ahead of the keys: the softmax asks for no more than scores)
              s_plan[pl] = s_tile[0][T % SLOTS] = word, s_in[0][T % SLOTS] = mask;
              if (both) s_tile[1][T1 % SLOTS] = word, s_in[1][T1 % SLOTS] = mask;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive_tc(plan_full + 8u * (uint32_t)pl);
            ++T, T1 += both;
          } while (once_more(word));
        }
        tiles += p.count();
      }
    } else {
      // ---- the products of row tile g
      const int g = warp - 16;
      const uint32_t id_s = idesc_h(128, TK, false), id_o = idesc_h(128, HD, true);
      const uint64_t dk = desc_k_tc(s0 + SM::K), dv = desc_mn_tc(s0 + SM::V, KBLK), dq = desc_k_tc(s0 + SM::Q + g * SM::QTILE);  // (steps are sums: in units of 16 bytes)
      int items = 0, tg = 0;  // items and tiles of this row tile
      int left = 0, ahead = 0;  // tiles of the piece of which scores are to be asked for; scores that are ahead of their product
      auto issue_s = [&]() {
        const int at = T + ahead, b = (tg + ahead) & 1;
        mbar_wait_short_tc(k_full + 8u * (uint32_t)(at % ST), (uint32_t)((at / ST) & 1), dead);
        __syncwarp();
        const int word = *(volatile int*)&s_tile[g][(tg + ahead) % SLOTS];  // (there when it is asked for, behind the instructions)
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (elect_tc()) {
          const uint64_t k = dk + (uint64_t)((at % ST) * (SM::TILE >> 4));
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk) {
            const uint64_t kd = k + (uint64_t)(((kk >> 2) * KBLK + (kk & 3) * 32) >> 4);
            if constexpr (SM::Q_TMEM) umma_ts_tc(t_s(g, b), t_q(g) + (uint32_t)(kk * 8), kd, id_s, kk != 0);
            else umma_tc(t_s(g, b), dq + (uint64_t)(((kk >> 2) * SM::QBLK + (kk & 3) * 32) >> 4), kd, id_s, kk != 0);
          }
          umma_commit_tc(bar_s + 16u * g + 8u * b);
          umma_commit_tc(k_free + 8u * (uint32_t)(at % ST));
        }
        __syncwarp();
        if (!once_more(word)) --left;
        ++ahead;
      };
      while (next_piece(p)) {
        left = p.count();
        if (g * 128 >= p.tokens * G) {  // nothing to do but to let the stages go
          for (; left > 0; ++T) {
            const uint32_t st = (uint32_t)(T % ST), ph = (uint32_t)((T / ST) & 1);
            mbar_wait_short_tc(k_full + 8u * st, ph, dead);
            __syncwarp();
            if (!once_more(*(volatile int*)&s_tile[0][T % SLOTS])) --left;
            if (lane == 0) mbar_arrive_tc(k_free + 8u * st);
            mbar_wait_short_tc(v_full + 8u * st, ph, dead);
            if (lane == 0) mbar_arrive_tc(v_free + 8u * st);
            __syncwarp();
          }
          continue;
        }
        mbar_wait_short_tc(bar_q + 8u * g, (uint32_t)(items & 1), dead);
        ++items;
#pragma unroll 1  // (every place that has these instructions costs the other roles some of theirs: written out twice 8192 rows took 581 us instead of 570)
        for (int k = 0; k < 2 && left > 0; ++k) issue_s();
        for (bool first = true; ahead > 0; first = false, --ahead, ++T, ++tg) {
          const uint32_t st = (uint32_t)(T % ST), ph = (uint32_t)((tg >> 1) & 1);
          const int b = tg & 1;
          mbar_wait_short_tc(v_full + 8u * st, (uint32_t)((T / ST) & 1), dead);
          mbar_wait_short_tc(bar_p + 16u * g + 8u * b, ph, dead);
          __syncwarp();
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          if (elect_tc()) {
            const uint64_t v = dv + (uint64_t)(st * (SM::TILE >> 4));
#pragma unroll
            for (int kk = 0; kk < TK / 16; ++kk) umma_ts_tc(t_o(g), t_s(g, b) + (uint32_t)(kk * 8), v + (uint64_t)(kk * 128), id_o, !first || kk > 0);
            umma_commit_tc(bar_o + 16u * g + 8u * b);
            umma_commit_tc(v_free + 8u * st);
          }
          __syncwarp();
          if (left > 0) {
            mbar_wait_short_tc(bar_o + 16u * g + 8u * b, ph, dead);  // the scores two tiles ahead go over the weights that this product reads
            issue_s();
          }
        }
      }
    }
  } else if (warp >= 8) {
    // ---- codes to fp16: keys by the first four warps, values by the others
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    constexpr int UNITS = TK * (HD / 16) / 128;  // 16 codes each, of a thread
    const int is_v = warp >= 12, w = warp & 3, r8 = lane & 7, cq = lane >> 3;
    // eight lanes side by side take the same columns of eight rows
    auto row_of = [&](int e) { return (HD == 128 ? e * 2 + (w & 1) : e * 4 + w) * 8 + r8; };
    const int piece = HD == 128 ? (w >> 1) * 4 + cq : cq, nb = piece / 4, c16 = (2 * piece) & 7;
    const uint32_t full = is_v ? v_full : k_full, free_ = is_v ? v_free : k_free;
    int R = 0;  // tiles as they are copied
    while (next_piece(p)) {
#pragma unroll 1
      for (int left = p.count(); left > 0; ++T) {
        const int rs = R % RAW, st = T % ST, pl = T % PLANS;
        mbar_wait_short_tc(raw_full + 8u * (uint32_t)rs, (uint32_t)((R / RAW) & 1), dead);
        const unsigned char* codes = smem + SM::C + (rs * 2 + is_v) * SM::CODES;
        uint4 code[UNITS];
#pragma unroll
        for (int e = 0; e < UNITS; ++e) {
          const int row = row_of(e);
          code[e] = *reinterpret_cast<const uint4*>(codes + piece_at<HD>(row, piece));
        }
        mbar_wait_short_tc(plan_full + 8u * (uint32_t)pl, (uint32_t)((T / PLANS) & 1), dead);
        const int word = *(volatile int*)&s_plan[pl];
        uint32_t factor[UNITS];
#pragma unroll
        for (int e = 0; e < UNITS; ++e) factor[e] = *(volatile uint32_t*)&s_factor[pl][is_v][row_of(e)];
        if (T >= ST) mbar_wait_short_tc(free_ + 8u * (uint32_t)st, (uint32_t)((T / ST - 1) & 1), dead);
        __syncwarp();
        const uint32_t to = s0 + (is_v ? SM::V : SM::K) + st * SM::TILE + nb * KBLK;
#pragma unroll
        for (int e = 0; e < UNITS; ++e) {
          const int row = row_of(e);
          const uint32_t f = factor[e];
          const uint4 c = code[e];
          uint32_t h[8];
          kv8_unpack<CODE>(c.x, h[0], h[1]), kv8_unpack<CODE>(c.y, h[2], h[3]), kv8_unpack<CODE>(c.z, h[4], h[5]), kv8_unpack<CODE>(c.w, h[6], h[7]);
#pragma unroll
          for (int j = 0; j < 8; ++j) h[j] = mul_h2(h[j], f);
          if (word & TILE_CLEAR) {
#pragma unroll
            for (int j = 0; j < 8; ++j) h[j] = f == CLEAR_H2 ? 0u : h[j];
          }
          const uint32_t line = to + row * 128;
          asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(line + ((c16 ^ r8) << 4)), "r"(h[0]), "r"(h[1]), "r"(h[2]), "r"(h[3]) : "memory");
          asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(line + (((c16 + 1) ^ r8) << 4)), "r"(h[4]), "r"(h[5]), "r"(h[6]), "r"(h[7]) : "memory");
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        const bool again = once_more(word);
        if (lane == 0) {
          mbar_arrive_tc(full + 8u * (uint32_t)st), mbar_arrive_tc(plan_free + 8u * (uint32_t)pl);
          if (!again) mbar_arrive_tc(raw_free + 8u * (uint32_t)rs);
        }
        if (!again) ++R, --left;
      }
    }
  } else {
    // ---- softmax: this thread's row
    asm volatile("setmaxnreg.inc.sync.aligned.u32 144;");
    const int g = warp >> 2, row = g * 128 + (tid & 127), tok = row / G, gh = row - tok * G;
    const uint32_t la = (uint32_t)((warp & 3) * 32) << 16;
    int tg = 0;  // tiles of this row tile
    if (tid == 0) info[blockIdx.x].parts = 0;
    bool more = next_piece(p);
    while (more) {
      const int rows = p.tokens * G;
      if (tid == 0 && !p.whole() && p.begin == 0)  // goes on in the CTAs behind; the item's last tile is at x1 - left + tiles - 1
        info[blockIdx.x] = JoinInfo{p.t0, p.tokens, p.kvh, (int)quotient(x1 - p.left + p.tiles - 1, share) - (int)blockIdx.x + 1};
      if (g * 128 >= rows) {
        more = next_piece(p);
        continue;
      }
      const bool mine = row < rows;
      // ---- the row's query
      float sl2;
      {
        const uint4* src = reinterpret_cast<const uint4*>(a.q + (size_t)(p.t0 + (mine ? tok : 0)) * a.q_stride + (size_t)(p.kvh * G + (mine ? gh : 0)) * HD);
        auto words = [&](int at, uint32_t (&x)[32]) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const uint4 v = mine ? src[at + j] : make_uint4(0, 0, 0, 0);
            x[4 * j] = v.x, x[4 * j + 1] = v.y, x[4 * j + 2] = v.z, x[4 * j + 3] = v.w;
          }
        };
        uint32_t x[32], most = 0;  // (64 elements at a time: the whole row would cost spills)
#pragma unroll
        for (int at = 0; at < HD / 8; at += 8) {
          words(at, x);
#pragma unroll
          for (int j = 0; j < 32; ++j) most = max(most, max(x[j] << 16 & 0x7fff0000u, x[j] & 0x7fff0000u));
        }
        float there, back;
        query_scale(most, there, back);
        sl2 = a.scale_log2 * back;
#pragma unroll
        for (int at = HD / 8 - 8; at >= 0; at -= 8) {
          if (at < HD / 8 - 8) words(at, x);
#pragma unroll
          for (int j = 0; j < 32; ++j) x[j] = pack_h(lo2f(x[j]) * there, hi2f(x[j]) * there);
          if constexpr (SM::Q_TMEM) {
            __syncwarp();
            tmem_st32_tc(t_q(g) + la + at * 4, x);
          } else {
            const uint32_t line = s0 + SM::Q + g * SM::QTILE + (at / 8) * SM::QBLK + (tid & 127) * 128;
#pragma unroll
            for (int j = 0; j < 8; ++j)
              asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(line + ((j ^ (tid & 7)) << 4)), "r"(x[4 * j]), "r"(x[4 * j + 1]), "r"(x[4 * j + 2]), "r"(x[4 * j + 3]) : "memory");
          }
        }
        if constexpr (SM::Q_TMEM) tmem_wait_st_tc();
        else asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        mbar_arrive_tc(bar_q + 8u * g);
      }
      const int my_pos = p.pos0 + min(tok, p.tokens - 1), my_low = a.window > 0 ? max(0, my_pos - a.window + 1) : 0;
      // the references of the row's weights, and beside that one (rel, a whole number) of its weights times the values' scales, of O; both of what the row sees
      float m_ref = -INFINITY, m_off = 0.f, rel = 0.f, l_run = 0.f;  // m_off: what is added to scores for it
      bool again;         // the tile
      bool huge = false;  // some row's reference is so large that scores round to fewer bits than their differences need
#pragma unroll 1
      for (int i = p.begin, first = 1; i < p.end; i += !again, first = 0, ++tg) {
        const int b = tg & 1;
        const uint32_t ts = t_s(g, b) + la, ph = (uint32_t)((tg >> 1) & 1);
        const int key = p.key0 + i * TK, last = my_pos - key, low = my_low - key;  // the first key of the tile; the last and the first that the row sees
        mbar_wait_short_tc(bar_s + 16u * g + 8u * b, ph, dead);
        __syncwarp();
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        uint32_t r[TK];
        tmem_ld32_tc(ts, r);
        tmem_ld32_tc(ts + 32, r + 32);
        const int tile = s_tile[g][tg % SLOTS];
        const float s = fmaxf(sl2 * __uint_as_float(tile & 0x7f800000u), 1e-37f), vt = __uint_as_float(0x4b000000u | (tile & 255)) - 8388735.f;  // (zero must not meet minus infinity; 2^23 + 127)
        tmem_wait_ld_tc();
        if (last < TK - 1 || low > 0 || tile & TILE_PART) {
          unsigned long long in = last < 0 || low >= TK ? 0 : ~0ull >> max(TK - 1 - last, 0) & ~0ull << max(low, 0);
          if (tile & TILE_PART) in &= s_in[g][tg % SLOTS];
          const uint32_t in0 = (uint32_t)in, in1 = (uint32_t)(in >> 32);
#pragma unroll
          for (int j = 0; j < TK; ++j)
            if (!((j < 32 ? in0 : in1) & 1u << (j & 31))) r[j] = 0xff800000u;  // -inf
        }
        float mx[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) mx[e] = max3_tc(__uint_as_float(r[e]), __uint_as_float(r[e + 4]), __uint_as_float(r[e + 8]));
#pragma unroll
        for (int j = 12; j + 8 <= TK; j += 8)
#pragma unroll
          for (int e = 0; e < 4; ++e) mx[e] = max3_tc(mx[e], __uint_as_float(r[j + e]), __uint_as_float(r[j + 4 + e]));
#pragma unroll
        for (int e = 0; e < 4; ++e) mx[e] = fmaxf(mx[e], __uint_as_float(r[60 + e]));
        const float top = __fmul_rn(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), s);
        const bool grow = __any_sync(0xffffffffu, ((top > m_ref + LAG || (top - m_ref) + vt > rel + LAG) && mine) || huge || tile & TILE_AGAIN);  // (one vote for all that is rare)
        float f = 1.f, sx = s;
        again = false;
        if (grow) {
          again = once_more(tile);
          const float m_new = fmaxf(m_ref, top);
          if (m_new > -INFINITY) {
            const float by = m_ref - m_new, before = rel + by, rel_new = fmaxf(floorf(before), ceilf((top - m_new) + vt));  // (nothing before: by minus infinity)
            l_run *= ex2_tc(by), f = ex2_tc(before - rel_new), rel = rel_new, m_ref = m_new, m_off = -m_new;
          }
          huge = __any_sync(0xffffffffu, fabsf(m_off) >= 4194304.f);
          if (huge) {  // the score rounded, as the maximum was, and then the difference (a packed product beside the packed sum would be fused with it)
#pragma unroll
            for (int j = 0; j < TK; j += 2) {
              float e0 = __fmul_rn(__uint_as_float(r[j]), s), e1 = __fmul_rn(__uint_as_float(r[j + 1]), s);
              add2_tc(e0, e1, m_off, m_off);
              r[j] = __float_as_uint(e0), r[j + 1] = __float_as_uint(e1);
            }
            sx = 1.f, m_off = 0.f;
          }
        }
        // weights by 2^7 and their values' scale beside the reference of those; 2^-64 of that is none in fp16, and one in the sum
        const float d = fmaxf(vt - rel, -64.f) + (float)P_EXP;
        const unsigned long long s2 = twice_tc(sx), n2 = twice_tc(m_off + d);
        float rs[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < TK; c += 32) {
          uint32_t wt[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float e0 = __uint_as_float(r[c + 2 * e]), e1 = __uint_as_float(r[c + 2 * e + 1]);
            fma2_tc(e0, e1, s2, n2);
            e0 = ex2_tc(e0), e1 = ex2_tc(e1);
            add2_tc(rs[2 * (e & 1)], rs[2 * (e & 1) + 1], e0, e1);
            wt[e] = pack_h(e0, e1);
          }
          tmem_st16_tc(ts + c / 2, wt);
        }
        l_run += ((rs[0] + rs[1]) + (rs[2] + rs[3])) * ex2_tc(-d);
        if (grow && !first) {  // O, behind the product of the tile before
          mbar_wait_short_tc(bar_o + 16u * g + 8u * (b ^ 1), (uint32_t)(((tg - 1) >> 1) & 1), dead);
          __syncwarp();
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
          for (int c = 0; c < HD; c += 64) {
            uint32_t o[64];
            tmem_ld32_tc(t_o(g) + la + c, o);
            tmem_ld32_tc(t_o(g) + la + c + 32, o + 32);
            tmem_wait_ld_tc();
#pragma unroll
            for (int j = 0; j < 64; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
            tmem_st32_tc(t_o(g) + la + c, o);
            tmem_st32_tc(t_o(g) + la + c + 32, o + 32);
          }
        }
        tmem_wait_st_tc();
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        mbar_arrive_tc(bar_p + 16u * g + 8u * b);
      }
      // ---- the row of the result, and (heads of 128) the next piece while the last product is under way: 8192 rows 586 -> 564 us; with heads of 64 16 portions 107 -> 108
      const bool whole = p.whole();
      bf16* dst = a.out + (size_t)(p.t0 + tok) * a.out_stride + (size_t)(p.kvh * G + gh) * HD;
      float* part = parts + ((size_t)blockIdx.x * 2 + (p.begin == 0)) * PART<HD, ROWS_P>;
      if (HD == 128) more = next_piece(p);
      mbar_wait_short_tc(bar_o + 16u * g + 8u * ((tg - 1) & 1), (uint32_t)(((tg - 1) >> 1) & 1), dead);
      __syncwarp();
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const float back = m_ref > -INFINITY ? result_scale(rel) : 0.f, nan = __int_as_float(0x7fc00000);
      const float scale = *dead ? nan : !whole ? back * (1 << LAG_EXP) : l_run > 0.f ? back * ((1 << LAG_EXP) / l_run) : l_run;
      if (!whole) part[ROWS_P * HD + row] = m_ref, part[ROWS_P * HD + ROWS_P + row] = *dead ? nan : l_run;
#pragma unroll
      for (int c = 0; c < HD; c += 32) {
        uint32_t r[32];
        __syncwarp();  // (the columns before end per thread)
        tmem_ld32_tc(t_o(g) + la + c, r);
        tmem_wait_ld_tc();
        if (mine && whole) {
#pragma unroll
          for (int j = 0; j < 32; j += 16) {
            uint32_t w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = pack2f(__uint_as_float(r[j + 2 * e]) * scale, __uint_as_float(r[j + 2 * e + 1]) * scale);
            if (out32) {
              asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(dst + c + j), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                           : "memory");
            } else {
              *reinterpret_cast<uint4*>(dst + c + j) = make_uint4(w[0], w[1], w[2], w[3]);
              *reinterpret_cast<uint4*>(dst + c + j + 8) = make_uint4(w[4], w[5], w[6], w[7]);
            }
          }
        } else if (mine) {
#pragma unroll
          for (int j = 0; j < 32; j += 4)
            *reinterpret_cast<float4*>(part + ((c + j) / 4 * ROWS_P + row) * 4) =
                make_float4(__uint_as_float(r[j]) * scale, __uint_as_float(r[j + 1]) * scale, __uint_as_float(r[j + 2]) * scale, __uint_as_float(r[j + 3]) * scale);
        }
      }
      __syncwarp();
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");  // (the next queries and weights let the products on)
      if (HD == 64) more = next_piece(p);
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 16) {
    drain_tc(dead);
    if (lane == 0) report_tc(dead, a.status);
    __syncwarp();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

template <int HD, int CODE, bool TMA>
cudaError_t launch_prompt(const BatchAttnArgs& a, const Kv8Geom& kv, int G, const TensorMap2D& cm, int box, cudaStream_t st) {
  static PerDeviceOnce set;
  if (set.need()) {
    const cudaError_t e = cudaFuncSetAttribute(attn_prompt8_kernel<HD, CODE, TMA>, cudaFuncAttributeMaxDynamicSharedMemorySize, SmemP<HD>::TOTAL);
    if (e != cudaSuccess) return e;
    set.done();
  }
  const int out32 = reinterpret_cast<uintptr_t>(a.out) % 32 == 0 && a.out_stride % 16 == 0;
  BatchAttnArgs b = a;
  b.rest = HD == 64 ? 5 : 8;  // (8192 rows, heads of 128, with 3: the CTAs that begin with a kv head's short items end at 680 us, the others at 555)
  return launched(launch_k(attn_prompt8_kernel<HD, CODE, TMA>, dim3(a.num_sms), dim3(THR_P), SmemP<HD>::TOTAL, st, b, kv, G, ROWS_P / G, out32, box,
                                          *reinterpret_cast<const CUtensorMap*>(&cm)));
}

// the parts of both kernels' items
template <int HD, int SLICES>
__global__ void __launch_bounds__(JOIN_THR, 2) attn_both8_join_kernel(BatchAttnArgs large, BatchAttnArgs small, JoinShape sh_large, JoinShape sh_small, int n_large, int n_small) {
  __shared__ Sum4 sums[JOIN_THR];
  pdl_wait();
  pdl_trigger();
  const int k = blockIdx.x;  // (of large items' columns parts side by side, and behind them small items)
  if (k < n_large * SLICES) join_parts<HD, ROWS_P>(large, sh_large, n_large, k / SLICES, k % SLICES, sums);
  else join_parts<HD, ROWS_F>(small, sh_small, n_small, k - n_large * SLICES, 0, sums);
}
size_t work_few(int hd, int num_sms) { return 2 * (size_t)num_sms * (sizeof(JoinInfo) + 2 * (hd == 64 ? PART<64, ROWS_F> : PART<128, ROWS_F>) * sizeof(float)); }
size_t work_prompt(int hd, int num_sms) { return (size_t)num_sms * (sizeof(JoinInfo) + 2 * (hd == 64 ? PART<64, ROWS_P> : PART<128, ROWS_P>) * sizeof(float)); }

}  // namespace

size_t attention_batch8_work(int hd, int num_sms) { return work_few(hd, num_sms) + work_prompt(hd, num_sms); }

cudaError_t launch_attention_batch8(const BatchAttnArgs& a, const Kv8Geom& kv, cudaStream_t st) {
  const int group = a.n_q / kv.n_kv, g = std::min(group, ROWS_F), P = kv.page_size;
  const JoinShape sh{g, group, (group + g - 1) / g};
  // Requests of at most 16 rows of a kv head are for blocks of few rows, which read their keys and values once to three times (once for each 16 heads of a larger group); the others have blocks
  // of up to 256 (a decode row in one of those costs what 256 rows do: 48 of them at 2800 positions on average beside four portions of a prompt 105 us, by both kernels 92; 16 portions without
  // decode rows 104 and 111, of which 6 are the kernel that finds nothing and begins when the other one has ended).  Where the step has no more rows than requests, all of them
  // are blocks of few rows (a request with many rows reads its keys and values that much more often); the room counts, which the host knows, and not the step's rows, which it does not.
  const bool few = a.n_tok <= a.n_req;
  // boxes of the most rows, a power of two, that divide a page and a unit or tile; a tile's scales come by bulk copies of a multiple of 16 bytes
  int box = 1;
  while (box < 64 && P % (2 * box) == 0) box *= 2;
  const int box_f = std::min(box, 32);
  const bool tma_f = box_f >= 4, tma_p = box >= 16 && (reinterpret_cast<uintptr_t>(kv.scale) & 15) == 0;
  const unsigned long long rows = (unsigned long long)kv.n_pages * kv.n_layers * 2ull * kv.n_kv * P;
  TensorMap2D cm_f{}, cm_p{};
  cudaError_t e = tma_f ? make_tensor_map_kv8(&cm_f, kv.codes, rows, kv.hd, box_f) : cudaSuccess;
  if (e == cudaSuccess && !few && tma_p) e = make_tensor_map_kv8(&cm_p, kv.codes, rows, kv.hd, box);
  if (e != cudaSuccess) return e;
  auto go = [&](auto hd, auto code) {
    constexpr int HD = decltype(hd)::value, CODE = decltype(code)::value;
    BatchAttnArgs small = a, large = a;
    if (!few) {
      small.n_most = large.n_more = ROWS_F / g;
      small.work = static_cast<char*>(a.work) + work_prompt(HD, a.num_sms);
      const cudaError_t r = tma_p ? launch_prompt<HD, CODE, true>(large, kv, group, cm_p, box, st) : launch_prompt<HD, CODE, false>(large, kv, group, cm_p, box, st);
      if (r != cudaSuccess) return r;
    }
    cudaError_t r;
    if (tma_f) r = group <= 8 ? launch_few<HD, CODE, 1, true>(small, kv, sh, 8 / g, box_f, !few, cm_f, st) : launch_few<HD, CODE, 2, true>(small, kv, sh, ROWS_F / g, box_f, !few, cm_f, st);
    else r = group <= 8 ? launch_few<HD, CODE, 1, false>(small, kv, sh, 8 / g, box_f, !few, cm_f, st) : launch_few<HD, CODE, 2, false>(small, kv, sh, ROWS_F / g, box_f, !few, cm_f, st);
    if (few || r != cudaSuccess) return r;
    constexpr int SLICES = HD / 4 / (JOIN_THR / ROWS_P) / 4;
    return launched(launch_k(attn_both8_join_kernel<HD, SLICES>, dim3((SLICES + 2) * a.num_sms), dim3(JOIN_THR), 0, st, large, small, JoinShape{group, group, 1}, sh, a.num_sms, 2 * a.num_sms));
  };
  using std::integral_constant;
  if (kv.hd == 64) return kv.code == KV8_E4M3 ? go(integral_constant<int, 64>(), integral_constant<int, KV8_E4M3>()) : go(integral_constant<int, 64>(), integral_constant<int, KV8_INT8>());
  return kv.code == KV8_E4M3 ? go(integral_constant<int, 128>(), integral_constant<int, KV8_E4M3>()) : go(integral_constant<int, 128>(), integral_constant<int, KV8_INT8>());
}

}  // namespace qie
