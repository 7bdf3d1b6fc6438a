// attn_batch_plan.cuh -- how attn_batch.cu shares out a step's work: the tiles of all requests, kv heads and blocks of rows, one after the other, are cut into
// equal stretches, one a CTA.  Host and device.
#pragma once
#include "kernels.h"

namespace qie {

constexpr int AB_TQ = 128, AB_TK = 64;  // rows (token x query head of the group) and keys of a tile
static_assert(AB_TK == 64, "floor_sum");
// What an item costs beside its tiles (queries in, the edge of what rows see, results out), in tiles: items of one tile take 3.6 us more than their tiles' 1.3.  (8192
// rows with 1: the CTA with the shortest items ends at 646 us, the mean at 536.)
constexpr int AB_REST = 3;

// sum over i < n of floor((a i + b) / 64), a >= 1.  With i = 64 q + r the term is a q + floor((a r + b) / 64), and over a whole period of r those add up to
// (63 (a - 1) + d - 1) / 2 + d floor(b / d), d = gcd(a, 64).
__host__ __device__ __forceinline__ long long floor_sum(unsigned n, unsigned a, unsigned b) {
  const unsigned q = n / 64, rest = n % 64, low = a & (0u - a), d = low < 64 ? low : 64;
  const long long period = (63ll * (a - 1) + d - 1) / 2 + (long long)(b & ~(d - 1));  // (d is a power of two)
  unsigned long long part = 0;
  const unsigned b0 = b % 64;
  unsigned at = b0, add = 0;
  for (unsigned r = 0; r < rest; ++r, at += a) add += at / 64;
  part = add + (unsigned long long)(b / 64) * rest;
  return (long long)q * period + 32ll * a * q * (q - 1ll) + (long long)a * q * rest + (long long)part;
}

// a request's rows: n of them behind c positions, in blocks of tt tokens; window 0: none
struct AbRequest {
  int n, c, nb;
};
// keys that rows of block b see: tiles [first, last)
__host__ __device__ __forceinline__ void ab_tiles(const AbRequest& r, int b, int tt, int window, int& first, int& last) {
  const long long row0 = (long long)b * tt, row1 = row0 + tt < r.n ? row0 + tt : r.n, low = window > 0 ? r.c + row0 - window + 1 : 0;
  first = low > 0 ? (int)(low / AB_TK) : 0;
  last = (int)((r.c + row1 + AB_TK - 1) / AB_TK);
}
// cost of the first x blocks
__host__ __device__ __forceinline__ long long ab_cost(const AbRequest& r, int x, int tt, int window, int rest = AB_REST) {
  if (x <= 0) return 0;
  const int full = x < r.nb ? x : r.nb - 1;
  long long sum = (long long)x * rest;
  if (full > 0) sum += floor_sum(full, tt, (unsigned)r.c + tt + AB_TK - 1);
  if (x == r.nb) sum += ((long long)r.c + r.n + AB_TK - 1) / AB_TK;
  if (window > 0) {
    const long long base = (long long)r.c - window + 1;
    const long long b0 = base >= 0 ? 0 : (-base + tt - 1) / tt;
    if (x > b0) sum -= floor_sum((unsigned)(x - b0), tt, (unsigned)(base + b0 * tt));
  }
  return sum;
}

// a request as the batch's arrays have it; n = 0: nothing to do, or values that make no sense
struct Raw {
  AbRequest r;
  int t0, slot;
};
__host__ __device__ __forceinline__ int ab_rest(const BatchAttnArgs& a) { return a.rest ? a.rest : AB_REST; }
__host__ __device__ __forceinline__ Raw request(const BatchAttnArgs& a, int i, int tt) {
  Raw w;
  const int t0 = a.q_start[i], t1 = a.q_start[i + 1], len = a.kv_len[i];
  w.slot = a.slots ? a.slots[i] : i;
  const bool ok = t0 >= 0 && t1 > t0 && t1 <= a.n_tok && t1 - t0 > a.n_more && (a.n_most == 0 || t1 - t0 <= a.n_most) && len >= t1 - t0 && len <= (long long)a.max_pages * a.kv.page_size && w.slot >= 0 && w.slot < a.max_seqs;
  w.t0 = t0;
  w.r.n = ok ? t1 - t0 : 0;
  w.r.c = ok ? len - w.r.n : 0;
  w.r.nb = (w.r.n + tt - 1) / tt;
  return w;
}
// a CTA's stretch of an item: tiles [begin, end) of its `tiles`, the first of which holds key `key0`
struct Piece {
  int t0, tokens, kvh, slot, pos0, key0, begin, end, tiles, limit;  // limit: positions of the item's request
  long long left;                                                    // of the CTA's stretch, with this piece
  __host__ __device__ int count() const { return end - begin; }
  __host__ __device__ bool whole() const { return begin == 0 && end == tiles; }
};
// the pieces of a CTA's stretch, in their order; every warp of a role walks them by itself
struct Walk {
  Raw w;
  int req, kvh, block, skip;
  long long left;
  __host__ __device__ bool next(const BatchAttnArgs& a, int tt, Piece& p) {
    for (;;) {
      if (left <= 0) return false;
      while (block >= w.r.nb) {  // the next head, or the next request that has rows
        block = 0;
        if (w.r.nb > 0 && ++kvh < a.kv.n_kv) break;
        kvh = 0;
        if (++req >= a.n_req) return false;
        w = request(a, req, tt);
      }
      int first, last;
      ab_tiles(w.r, block, tt, a.window, first, last);
      const int tiles = last - first;
      const bool some = skip < tiles;
      if (some) {
        p.left = left;
        p.begin = skip;
        p.end = skip + left < tiles ? (int)(skip + left) : tiles;
        p.tiles = tiles;
        p.key0 = first * AB_TK;
        p.kvh = kvh;
        p.slot = w.slot;
        p.t0 = w.t0 + block * tt;
        p.tokens = w.r.n - block * tt < tt ? w.r.n - block * tt : tt;
        p.pos0 = w.r.c + block * tt;
        p.limit = w.r.c + w.r.n;
      }
      left -= tiles + ab_rest(a) - skip;
      skip = 0;
      ++block;
      if (some) return true;
    }
  }
};

}  // namespace qie
