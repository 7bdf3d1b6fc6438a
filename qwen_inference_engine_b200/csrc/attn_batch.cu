// attn_batch.cu -- attention of a step's rows over the paged cache on tcgen05 / TMEM: requests with any number of rows, causal behind their cached positions,
// with an optional window (qie_attention_batch).
//
//   out_t = sum_j 2^(s (q_t . k_j) - m) v_j / sum_j 2^(s (q_t . k_j) - m) over the positions j that row t sees, m their running maximum
//
// An item is a kv head of a request and a block of its tokens: the rows of a tile are (token, query head of the group), so keys and values are read once
// for the whole group and a decode row costs the tiles of its context alone.  The tiles of all items, one after the other, are cut into equal stretches,
// one a CTA (two CTAs an SM; the host knows no lengths, so every CTA adds the requests up itself).  An item that is cut leaves its parts (rows of O, maximum,
// sum, in fp32) in the work area, and a second kernel joins them, in their order.  (Joined by the CTA that comes last: no quicker for a single row, 10.4 us as with the
// kernel, as what another SM wrote is as far away as the start of a kernel; and 10 us for 126 rows.)
// Within a CTA:
//   S = Q K^T  : tcgen05.mma, 128 x 64 fp32 in one of two TMEM buffers, issued two tiles ahead of its softmax, across items
//   softmax    : warps 0-3, a thread a row (= TMEM lane).  The weights go back over the scores as bf16: the product's A operand (2^-8 of each weight; sums take
//                them unrounded).  Warps without rows only pass the barriers on.
//   O += P V   : accumulates in TMEM; rows scale it when their maximum grows by more than LAG
//   warp 4     : the products.  warp 5: queries and 64-column boxes of the pages by TMA with the 128-byte swizzle, or, for pages of other than multiples of 16
//                positions, 16-byte copies to the same places.
// Values of keys that some row of a tile does not see must not meet its zero weight when they are no numbers: tiles at the edges of what rows see are
// looked over, such values are put aside, and rows that see them get them at the end.
// What bounds it (B200).  Prompts: the chain of a tile (scores, softmax, product), of which an SM has two under way: tensor pipe 52 % busy, exponentials 53 %, issue 40 %, L2
// 34 %; 8192 rows of 28 heads of 128 on 4 take 486 us, 990 TFLOP/s, for 10 ms at 1.96 GHz, and 552 us under the power cap at 1.7 (beside 500 in a run of 0.1 s: without exponentials 486, with half of the keys' and values' bytes 447, one CTA an SM 940).  Decode rows: DRAM, 6.2 TB/s between the first tiles and the last: 64 rows at 1434 positions on average, 189 MB, take 42.2 us, of
// which 7 us pass before the first scores and 6 behind the last tile.  One row behind 700 positions: 9.3 us, a chain of latencies (plan 1.3, pages and keys 2.4, a tile 0.8, its
// product and results 1.2, the start of the second kernel 1.2, joining 2.0).
// Every wait has a limit; when one runs out the CTA's results are not numbers and it reports it.
#include <cuda.h>

#include <algorithm>
#include <type_traits>

#include "attn_batch_split.cuh"
#include "common.cuh"
#include "kernels.h"
#include "launch.h"
#include "pack.cuh"
#include "tc_ptx.cuh"

namespace qie {
namespace {

constexpr int TQ = AB_TQ, TK = AB_TK;
constexpr int KBLK = TK * 128;  // [rows][64 columns] bf16 in 8-row swizzle atoms
constexpr int NSOFT = 128, NTHR = NSOFT + 64;
constexpr uint32_t TMEM_COLS = 256;  // two tiles of scores, O
// The weights' reference follows a row's maximum where it has fallen behind by more than this (powers of two), so that most tiles leave O as it is.  It costs exactness: the largest
// weight is then one no longer, and rounded like the others, by 2^-8 of itself at most (sums are fp32).  8192 rows, time beside that with 8 and error beside that of a result which is
// only rounded at its end: no lag 1.09 and 1.20, by 1 1.07 and 1.22, by 3 1.01 and 1.27, by 8 1.32.  Blocks of one token have none: 64 decode rows 42.2 us instead of 41.9
// and 1.23 instead of 1.38.
constexpr float LAG = 3.f;

// FEW: blocks of at most 16 rows (decode rows).  The products read 128 all the same, what lies behind their queries, and nobody looks at what comes of it; the room that the other
// queries would take is a third stage of keys and values (head size 64: a fifth and sixth): 64 rows at 2048 43.6 us, so 41.8.
template <int HD, bool FEW>
struct Smem {
  static constexpr int ROWS = FEW ? 16 : TQ, QBLK = ROWS * 128;
  // tiles of an item at the edges of what its rows see: tokens span at most 128 positions, so three at either end (16: two)
  static constexpr int EDGES = FEW ? 4 : 6;
  static constexpr int NB = HD / 64, ST = HD == 64 ? (FEW ? 6 : 4) : (FEW ? 3 : 2);  // column blocks; stages of K and of V
  static constexpr int TILE = NB * KBLK;
  static constexpr int Q = 0, K = NB * QBLK, V = K + ST * TILE, ODD = V + ST * TILE, BAR = ODD + EDGES * HD * 16, END = BAR + 512 + 1024;
  // (three CTAs an SM would wait for TMEM columns: see attn_prompt_tc.cu)
  static constexpr int TOTAL = END > 76 * 1024 ? END : 76 * 1024;
  static_assert(512 / TMEM_COLS == 2 && 3 * (TOTAL + 1024) > 228 * 1024 && 2 * (TOTAL + 2048) <= 228 * 1024, "two CTAs an SM");
};
struct Shape {
  int g, tt, out32;  // query heads of a group; tokens of a block; rows of the result begin on 32-byte boundaries
};
template <int HD, bool TMA, bool FEW>
__global__ void __launch_bounds__(NTHR, 2) attn_batch_kernel(BatchAttnArgs a, Shape sh, int box, const __grid_constant__ CUtensorMap qm, const __grid_constant__ CUtensorMap kvm) {
  using SM = Smem<HD, FEW>;
  constexpr int NB = SM::NB, ST = SM::ST, QBLK = SM::QBLK, EDGES = SM::EDGES;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  __shared__ long long s_sums[NTHR / 32];
  __shared__ Walk s_walk;
  __shared__ int dead_s, s_odd[2], s_edge[EDGES];  // s_odd, by the item's parity: there are values put aside; s_edge: first keys of the edge tiles
  volatile int* dead = &dead_s;
  if (threadIdx.x == NTHR - 1) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&qm) : "memory");
    if (TMA) asm volatile("prefetch.tensormap [%0];" ::"l"(&kvm) : "memory");
  }
  pdl_wait();
  pdl_trigger();
  const uint32_t s0 = (smem_u32(smem_raw) + 1023u) & ~1023u;
  // barriers: of S, P and O in pairs by the tile's parity; of the queries and of K and V a stage each, full and free
  const uint32_t bar_s = s0 + SM::BAR, bar_p = bar_s + 16, bar_o = bar_s + 32, bar_q = bar_s + 48, slot = bar_s + 56, bar_k = bar_s + 64, bar_v = bar_k + 8 * ST,
                 free_k = bar_v + 8 * ST, free_v = free_k + 8 * ST, free_q = free_v + 8 * ST;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, tt = sh.tt, G = sh.g;
  if (tid == 0) {
    dead_s = 0, s_odd[0] = s_odd[1] = 0, s_walk.left = 0;
    for (int i = 0; i < 2; ++i) mbar_init_tc(bar_s + 8 * i, 1), mbar_init_tc(bar_p + 8 * i, NSOFT), mbar_init_tc(bar_o + 8 * i, 1);
    mbar_init_tc(bar_q, 1), mbar_init_tc(free_q, 1);
    for (int i = 0; i < ST; ++i) mbar_init_tc(bar_k + 8 * i, 1), mbar_init_tc(bar_v + 8 * i, 1), mbar_init_tc(free_k + 8 * i, 1), mbar_init_tc(free_v + 8 * i, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == NSOFT / 32) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  for (int i = tid; i < EDGES * HD; i += NTHR) asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(s0 + SM::ODD + i * 16), "r"(0u) : "memory");
  const auto [share, x1] = find_stretch<NTHR>(a, tt, s_sums, &s_walk);
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  Walk walk = s_walk;
  uint32_t tmem;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem) : "r"(slot));
  const uint32_t t_o = tmem + 128;  // scores: columns 0 .. 63 and 64 .. 127, the weights over them
  JoinInfo* info = reinterpret_cast<JoinInfo*>(a.work);
  unsigned long long* odd_bits = reinterpret_cast<unsigned long long*>(smem_raw + (s0 - smem_u32(smem_raw)) + SM::ODD);  // [edge tile][column][2]
  float* parts = reinterpret_cast<float*>(info + gridDim.x);

  if (warp == NSOFT / 32 + 1) {
    // ---- copies
    const int P = a.kv.page_size, chunks = TK / box;  // of a tile
    const uint32_t q_bytes = (uint32_t)(NB * tt * G * 128);
    const int none = a.kv.n_pages * a.kv.n_layers * 2 * a.kv.n_kv * P;  // (TMA) a row behind the pool: zeros
    Piece p;
    int T = 0;  // tiles so far
    for (int item = 0; walk.next(a, tt, p); ++item) {
      const int* bt = a.block_table + (size_t)p.slot * a.max_pages;
      const int last_page = (p.limit - 1) / P;
      const int c0 = p.key0 / box;  // chunks of `box` keys; a lane holds the page of chunk `held` + lane
      int held = c0 + p.begin * chunks, page_of = 0;
      if (TMA) page_of = bt[min((held + lane) * box / P, last_page)];  // chunks behind the last page repeat it (their keys are masked)
      if (item > 0) mbar_wait_tc(free_q, (uint32_t)((item - 1) & 1), dead);
      if (lane == 0) asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar_q), "r"(q_bytes) : "memory");
      __syncwarp();
      if (lane < NB)
        asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                     ::"r"(s0 + SM::Q + lane * QBLK), "l"(&qm), "r"(bar_q), "r"(lane * 64), "r"(p.kvh * G), "r"(p.t0)
                     : "memory");
      __syncwarp();
      for (int i = p.begin; i < p.end; ++i, ++T) {
        const uint32_t st = (uint32_t)(T % ST);
        if constexpr (TMA) {
          const int ch = c0 + i * chunks;
          if (ch + chunks > held + 32) {
            held = ch;
            page_of = bt[min((held + lane) * box / P, last_page)];
          }
          const int j = lane / NB, nb = lane % NB, page = __shfl_sync(0xffffffffu, page_of, (ch - held + j) & 31);
          const int at = min((ch + j) * box, last_page * P + P - box) % P;  // (positions end at 2^30)
          const bool in = page >= 0 && page < a.kv.n_pages;
#pragma unroll
          for (int is_v = 0; is_v < 2; ++is_v) {
            if (T >= ST) mbar_wait_tc((is_v ? free_v : free_k) + 8u * st, (uint32_t)((T / ST - 1) & 1), dead);
            const uint32_t bar = (is_v ? bar_v : bar_k) + 8u * st, dst = s0 + (is_v ? SM::V : SM::K) + st * SM::TILE + nb * KBLK + j * box * 128;
            const int row = in ? (((page * a.kv.n_layers + a.layer) * 2 + is_v) * a.kv.n_kv + p.kvh) * P + at : none;
            if (lane == 0) asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"((uint32_t)SM::TILE) : "memory");
            __syncwarp();
            if (lane < chunks * NB)
              asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                           ::"r"(dst), "l"(&kvm), "r"(bar), "r"(nb * 64), "r"(row)
                           : "memory");
            __syncwarp();
          }
        } else {
#pragma unroll
          for (int is_v = 0; is_v < 2; ++is_v) {
            if (T >= ST) mbar_wait_tc((is_v ? free_v : free_k) + 8u * st, (uint32_t)((T / ST - 1) & 1), dead);
            const uint32_t dst = s0 + (is_v ? SM::V : SM::K) + st * SM::TILE;
            const int c = lane & 7;
            for (int k = lane >> 3; k < TK; k += 4) {  // eight lanes a row
              const int key = min(p.key0 + i * TK + k, p.limit - 1), pg = key / P, page = bt[pg];
              const bool in = page >= 0 && page < a.kv.n_pages;
              const bf16* src = a.kv.chunk(in ? page : 0, a.layer, is_v, p.kvh) + (size_t)(key - pg * P) * HD + c * 8;
#pragma unroll
              for (int nb = 0; nb < NB; ++nb) cp_async16(dst + nb * KBLK + k * 128 + ((c ^ (k & 7)) << 4), src + nb * 64);
            }
            cp_async_commit();
            cp_async_wait<0>();
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive_tc((is_v ? bar_v : bar_k) + 8u * st);
          }
        }
      }
    }
  } else if (warp == NSOFT / 32) {
    // ---- products
    const uint32_t id_s = idesc_tc(TQ, TK, false), id_o = idesc_tc(TQ, HD, true);
    const uint64_t dq = desc_k_tc(s0 + SM::Q), dk = desc_k_tc(s0 + SM::K), dv = desc_mn_tc(s0 + SM::V, KBLK);  // (steps are sums: in units of 16 bytes)
    Walk ahead = walk;
    Piece p;
    int TS = 0, s_left = 0, items = 0;  // tiles of S issued; of the item they are in, left; items begun
    auto issue_s = [&]() {              // the next tile's scores, if there is one
      if (s_left == 0) {
        Piece n;
        if (!ahead.next(a, tt, n)) {
          s_left = -1;
          return;
        }
        s_left = n.count();
        mbar_wait_tc(bar_q, (uint32_t)(items & 1), dead);
        ++items;
      }
      if (s_left < 0) return;
      const uint64_t k = dk + (uint64_t)((TS % ST) * (SM::TILE >> 4));
      mbar_wait_tc(bar_k + 8u * (uint32_t)(TS % ST), (uint32_t)((TS / ST) & 1), dead);
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      if (elect_tc()) {
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk)
          umma_tc(tmem + (uint32_t)((TS & 1) * TK), dq + (uint64_t)(((kk >> 2) * QBLK + (kk & 3) * 32) >> 4), k + (uint64_t)(((kk >> 2) * KBLK + (kk & 3) * 32) >> 4), id_s,
                  kk != 0);
        umma_commit_tc(bar_s + 8u * (uint32_t)(TS & 1));
        umma_commit_tc(free_k + 8u * (uint32_t)(TS % ST));
        if (s_left == 1) umma_commit_tc(free_q);
      }
      __syncwarp();
      ++TS, --s_left;
    };
    issue_s();
    issue_s();
    for (int T = 0; walk.next(a, tt, p);)
      for (int i = 0; i < p.count(); ++i, ++T) {
        const uint32_t b = 8u * (uint32_t)(T & 1), ph = (uint32_t)((T >> 1) & 1), st = (uint32_t)(T % ST);
        mbar_wait_tc(bar_v + 8u * st, (uint32_t)((T / ST) & 1), dead);
        mbar_wait_tc(bar_p + b, ph, dead);
        const uint32_t w = tmem + (uint32_t)((T & 1) * TK);
        const uint64_t v = dv + (uint64_t)(st * (SM::TILE >> 4));
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (elect_tc()) {
#pragma unroll
          for (int kk = 0; kk < TK / 16; ++kk) umma_ts_tc(t_o, w + (uint32_t)(kk * 8), v + (uint64_t)(kk * 128), id_o, i > 0 || kk > 0);
          umma_commit_tc(bar_o + b);
          umma_commit_tc(free_v + 8u * st);
        }
        __syncwarp();
        if (s_left >= 0) {
          mbar_wait_tc(bar_o + b, ph, dead);  // S(T + 2) goes over the weights that P V(T) reads
          issue_s();
        }
      }
  } else {
    // ---- softmax: this thread's row
    const int row = tid, tok = row / G, g = row - tok * G;
    const uint32_t la = (uint32_t)(warp * 32) << 16;
    const float sl2 = a.scale_log2;
    Piece p;
    int T = 0;
    if (tid == 0) info[blockIdx.x].parts = 0;
    for (int item = 0; walk.next(a, tt, p); ++item) {
      const bool some = warp * 32 < p.tokens * G;  // the warp has rows
      const int my_pos = p.pos0 + min(tok, p.tokens - 1), my_low = a.window > 0 ? max(0, my_pos - a.window + 1) : 0;
      const int low0 = a.window > 0 ? max(0, p.pos0 - a.window + 1) : 0, low1 = a.window > 0 ? max(0, p.pos0 + p.tokens - a.window) : 0;  // of the first and the last token
      const float lag = p.tokens > 1 ? LAG : 0.f;
      float m_ref = -INFINITY, l_run = 0.f;
      int edge = 0;
      for (int i = p.begin; i < p.end; ++i, ++T) {
        const uint32_t b = 8u * (uint32_t)(T & 1), ph = (uint32_t)((T >> 1) & 1), ts = tmem + la + (uint32_t)((T & 1) * TK), st = (uint32_t)(T % ST);
        const int key = p.key0 + i * TK, last = my_pos - key, low = my_low - key;  // the first key of the tile; the last and the first that the row sees
        mbar_wait_warp_tc(bar_s + b, ph, dead);
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (some) {
          uint32_t r[64];
          tmem_ld32_tc(ts, r);
          tmem_ld32_tc(ts + 32, r + 32);
          tmem_wait_ld_tc();
          if (last < TK - 1) {
#pragma unroll
            for (int j = 0; j < TK; ++j)
              if (j > last) r[j] = 0xff800000u;  // -inf
          }
          if (low > 0) {
#pragma unroll
            for (int j = 0; j < TK; ++j)
              if (j < low) r[j] = 0xff800000u;
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
          const float m_new = fmaxf(m_ref, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * sl2);
          const bool grow = __any_sync(0xffffffffu, m_new > m_ref + lag && tok < p.tokens);  // (rows behind the last token are anything)
          const float f = grow && m_new > -INFINITY ? ex2_tc(m_ref - m_new) : 1.f;
          if (grow) m_ref = m_new;
          const unsigned long long s2 = twice_tc(sl2), n2 = twice_tc(m_ref > -INFINITY ? -m_ref : 0.f);
          float rs[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c = 0; c < TK; c += 32) {
            uint32_t w[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              float e0 = __uint_as_float(r[c + 2 * e]), e1 = __uint_as_float(r[c + 2 * e + 1]);
              fma2_tc(e0, e1, s2, n2);
              e0 = ex2_tc(e0), e1 = ex2_tc(e1);
              add2_tc(rs[2 * (e & 1)], rs[2 * (e & 1) + 1], e0, e1);
              w[e] = pack2f(e0, e1);
            }
            tmem_st16_tc(ts + c / 2, w);
          }
          l_run = l_run * f + ((rs[0] + rs[1]) + (rs[2] + rs[3]));
          if (grow && i > p.begin) {  // scale O by the new reference; behind the exponentials the product of the tile before is in
            mbar_wait_warp_tc(bar_o + (b ^ 8u), (uint32_t)(((T - 1) >> 1) & 1), dead);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
            for (int c = 0; c < HD; c += 64) {
              uint32_t o[64];
              tmem_ld32_tc(t_o + la + c, o);
              tmem_ld32_tc(t_o + la + c + 32, o + 32);
              tmem_wait_ld_tc();
#pragma unroll
              for (int j = 0; j < 64; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
              tmem_st32_tc(t_o + la + c, o);
              tmem_st32_tc(t_o + la + c + 32, o + 32);
            }
          }
        }
        if ((key + TK > p.pos0 + 1 || key < low1) && edge < EDGES) {  // some row does not see some key of the tile
          mbar_wait_tc(bar_v + 8u * st, (uint32_t)((T / ST) & 1), dead);
          if (tid == 0) s_edge[edge] = key;
          for (int e = tid; e < TK * NB * 8; e += NSOFT) {
            const int nb = e / (TK * 8), k = (e >> 3) & (TK - 1), c = e & 7, at = key + k;
            const uint32_t addr = s0 + SM::V + st * SM::TILE + (uint32_t)(nb * KBLK + k * 128 + (c << 4));
            uint32_t x[4];
            asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(addr));
            bool odd = false;
#pragma unroll
            for (int y = 0; y < 4; ++y) odd |= (x[y] & 0x7f80u) == 0x7f80u || (x[y] & 0x7f800000u) == 0x7f800000u;
            if (!odd) continue;
            if (at >= p.pos0 + p.tokens || at < low0) {  // no row of the item sees the key
              x[0] = x[1] = x[2] = x[3] = 0;
            } else {
              s_odd[item & 1] = 1;
#pragma unroll
              for (int y = 0; y < 8; ++y) {
                const uint32_t v = (y & 1 ? x[y >> 1] >> 16 : x[y >> 1]) & 0xffffu;
                if ((v & 0x7f80u) != 0x7f80u) continue;
                x[y >> 1] &= y & 1 ? 0xffffu : 0xffff0000u;
                // a bit a key: in the first word +infinity, in the second -infinity, in both no number
                unsigned long long* to = odd_bits + 2 * (edge * HD + nb * 64 + ((c ^ (k & 7)) << 3) + y);
                if (v != 0xff80u) atomicOr(to, 1ull << k);
                if (v != 0x7f80u) atomicOr(to + 1, 1ull << k);
              }
            }
            asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]) : "memory");
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          ++edge;
          __syncwarp();  // (the loop above ends per thread, and what follows wants the warp's threads together)
        }
        tmem_wait_st_tc();
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        mbar_arrive_tc(bar_p + b);
      }
      // ---- the item's rows
      mbar_wait_warp_tc(bar_o + 8u * (uint32_t)((T - 1) & 1), (uint32_t)(((T - 1) >> 1) & 1), dead);
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const bool whole = p.whole();
      const int odd = *(volatile int*)&s_odd[item & 1];  // (a thread may be in the next item already, none in the one behind it)
      if (some) {
        const float scale = *dead ? __int_as_float(0x7fc00000) : !whole ? 1.f : l_run > 0.f ? 1.f / l_run : l_run;
        bf16* dst = a.out + (size_t)(p.t0 + tok) * a.out_stride + (size_t)(p.kvh * G + g) * HD;
        float* part = parts + ((size_t)blockIdx.x * 2 + (p.begin == 0)) * PART<HD, TQ>;
        if (!whole) part[TQ * HD + row] = m_ref, part[TQ * HD + TQ + row] = *dead ? __int_as_float(0x7fc00000) : l_run;
#pragma unroll
        for (int c = 0; c < HD; c += 32) {
          uint32_t r[32];
          __syncwarp();  // (the columns before end per thread)
          tmem_ld32_tc(t_o + la + c, r);
          tmem_wait_ld_tc();
          if (odd)
            for (int n = 0; n < edge; ++n) {
              // the keys of the edge tile that the row sees
              const int from = max(0, my_low - s_edge[n]), to = min(TK - 1, my_pos - s_edge[n]);
              const unsigned long long sees = from > to ? 0ull : (~0ull >> (TK - 1 - to)) & (~0ull << from);
#pragma unroll
              for (int j = 0; j < 32; ++j) {
                const unsigned long long* bits = odd_bits + 2 * (n * HD + c + j);
                if (bits[0] & sees) r[j] = __float_as_uint(__uint_as_float(r[j]) + INFINITY);
                if (bits[1] & sees) r[j] = __float_as_uint(__uint_as_float(r[j]) - INFINITY);
              }
            }
          if (tok < p.tokens && whole) {
#pragma unroll
            for (int j = 0; j < 32; j += 16) {
              uint32_t w[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) w[e] = pack2f(__uint_as_float(r[j + 2 * e]) * scale, __uint_as_float(r[j + 2 * e + 1]) * scale);
              if (sh.out32) {
                asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(dst + c + j), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                             : "memory");
              } else {
                *reinterpret_cast<uint4*>(dst + c + j) = make_uint4(w[0], w[1], w[2], w[3]);
                *reinterpret_cast<uint4*>(dst + c + j + 8) = make_uint4(w[4], w[5], w[6], w[7]);
              }
            }
          } else if (tok < p.tokens) {
#pragma unroll
            for (int j = 0; j < 32; j += 4) *reinterpret_cast<uint4*>(part + ((c + j) / 4 * TQ + row) * 4) = make_uint4(r[j], r[j + 1], r[j + 2], r[j + 3]);
          }
        }
      }
      if (tid == 0 && !whole && p.begin == 0)  // goes on in the CTAs behind; the item's last tile is at x1 - left + tiles - 1
        info[blockIdx.x] = JoinInfo{p.t0, p.tokens, p.kvh, (int)quotient(x1 - p.left + p.tiles - 1, share) - (int)blockIdx.x + 1};
      if (odd) {  // the same in every thread: arrivals at bar_p lie between the writes and this
        asm volatile("bar.sync 1, 128;" ::: "memory");
        for (int e = tid; e < EDGES * HD; e += NSOFT) odd_bits[2 * e] = odd_bits[2 * e + 1] = 0;
        if (tid == 0) s_odd[item & 1] = 0;
        asm volatile("bar.sync 1, 128;" ::: "memory");
      }
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == NSOFT / 32) {
    drain_tc(dead);
    if (lane == 0) report_tc(dead, a.status);
    __syncwarp();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
  }
}

template <int HD, bool TMA, bool FEW>
cudaError_t launch_hd(const BatchAttnArgs& a, int tt, const TensorMap2D& qm, const TensorMap2D& kvm, int box, cudaStream_t st) {
  static PerDeviceOnce set;
  if (set.need()) {
    const cudaError_t e = cudaFuncSetAttribute(attn_batch_kernel<HD, TMA, FEW>, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<HD, FEW>::TOTAL);
    if (e != cudaSuccess) return e;
    set.done();
  }
  const int G = a.n_q / a.kv.n_kv, ctas = 2 * a.num_sms;
  const cudaError_t e = launched(launch_k(attn_batch_kernel<HD, TMA, FEW>, dim3(ctas), dim3(NTHR), Smem<HD, FEW>::TOTAL, st, a, Shape{G, tt, (int)(reinterpret_cast<uintptr_t>(a.out) % 32 == 0 && a.out_stride % 16 == 0)}, box,
                                          *reinterpret_cast<const CUtensorMap*>(&qm), *reinterpret_cast<const CUtensorMap*>(&kvm)));
  if (e != cudaSuccess) return e;
  return launch_join<HD, TQ>(a, JoinShape{G, G, 1}, ctas, st);
}

}  // namespace

size_t attention_batch_work(int hd, int num_sms) { return (size_t)2 * num_sms * (sizeof(JoinInfo) + 2 * (hd == 64 ? PART<64, TQ> : PART<128, TQ>) * sizeof(float)); }

cudaError_t launch_attention_batch(const BatchAttnArgs& a, cudaStream_t st) {
  const int G = a.n_q / a.kv.n_kv, P = a.kv.page_size;
  const unsigned long long rows = (unsigned long long)a.kv.n_pages * a.kv.n_layers * 2ull * a.kv.n_kv * P;
  const bool tma = P % 16 == 0;
  // No more rows than requests: a decode step, or nearly one (a request with several rows has blocks of fewer of them, and reads its keys and values that much more often).
  // Else blocks of as many rows as the products take: one portion of 8192 rows of 7 heads a group has 456 blocks instead of 4096.  Rows behind 2000 positions, groups of 7,
  // room for as many rows as requests and for one more: 64 requests of a row 53.2 and 55.2 us (heads of 64: 23.9 both), 32 of two 33.1 and 34.4 (16.8, 16.9), 8 of eight 27.1 and
  // 23.1 (17.1, 22.8), one of 64 27.5 and 31.5 (17.5, 37.1).  The room counts, not the step's rows, which the host does not know: a graph with room for more rows than requests takes
  // large blocks in its decode steps too.
  const bool few = tma && G <= 16 && a.n_tok <= a.n_req;
  const int tt = (few ? 16 : TQ) / G;
  TensorMap2D qm, kvm{};
  cudaError_t e = make_tensor_map_heads(&qm, a.q, a.kv.hd, a.n_q, a.n_tok, a.q_stride, G, tt);
  if (e != cudaSuccess) return e;
  const int box = !tma ? TK : P % 64 == 0 ? 64 : P % 32 == 0 ? 32 : 16;  // the largest that divides a page and a tile
  if (tma && (e = make_tensor_map_kv(&kvm, a.kv.pool, rows, a.kv.hd, box)) != cudaSuccess) return e;
  if (a.kv.hd == 64)
    return few ? launch_hd<64, true, true>(a, tt, qm, kvm, box, st) : tma ? launch_hd<64, true, false>(a, tt, qm, kvm, box, st) : launch_hd<64, false, false>(a, tt, qm, kvm, box, st);
  return few ? launch_hd<128, true, true>(a, tt, qm, kvm, box, st) : tma ? launch_hd<128, true, false>(a, tt, qm, kvm, box, st) : launch_hd<128, false, false>(a, tt, qm, kvm, box, st);
}

}  // namespace qie
