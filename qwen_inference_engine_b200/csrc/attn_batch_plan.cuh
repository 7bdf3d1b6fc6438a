// attn_batch_plan.cuh -- how attn_batch.cu shares out a step's work: the tiles of all requests, kv heads and blocks of rows, one after the other, are cut into
// equal stretches, one a CTA.  Host and device.
#pragma once
#include "kernels.h"

namespace qie {

constexpr int AB_TQ = 128, AB_TK = 64;  // rows (token x query head of the group) and keys of a tile
constexpr int AB_REST = 1;              // what an item costs beside its tiles (queries in, results out), in tiles

// sum over i < n of floor((a i + b) / m), by the steps of Euclid's algorithm (a and m change places): n < 2^24, a <= 128, m = 64, b < 2^32
__host__ __device__ __forceinline__ long long floor_sum(unsigned n, unsigned m, unsigned a, unsigned b) {
  long long sum = 0;
  for (;;) {
    if (a >= m) sum += (long long)n * (n - 1) / 2 * (a / m), a %= m;
    if (b >= m) sum += (long long)n * (b / m), b %= m;
    const unsigned y = a * n + b;  // below 64 * 2^24 + 64
    if (y < m) return sum;
    n = y / m, b = y % m;
    const unsigned t = m;
    m = a, a = t;
  }
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
__host__ __device__ __forceinline__ long long ab_cost(const AbRequest& r, int x, int tt, int window) {
  if (x <= 0) return 0;
  const int full = x < r.nb ? x : r.nb - 1;
  long long sum = (long long)x * AB_REST;
  if (full > 0) sum += floor_sum(full, AB_TK, tt, (unsigned)r.c + tt + AB_TK - 1);
  if (x == r.nb) sum += ((long long)r.c + r.n + AB_TK - 1) / AB_TK;
  if (window > 0) {
    const long long base = (long long)r.c - window + 1;
    const long long b0 = base >= 0 ? 0 : (-base + tt - 1) / tt;
    if (x > b0) sum -= floor_sum((unsigned)(x - b0), AB_TK, tt, (unsigned)(base + b0 * tt));
  }
  return sum;
}

// a request as the batch's arrays have it; n = 0: nothing to do, or values that make no sense
struct Raw {
  AbRequest r;
  int t0, slot;
};
__host__ __device__ __forceinline__ Raw request(const BatchAttnArgs& a, int i, int tt) {
  Raw w;
  const int t0 = a.q_start[i], t1 = a.q_start[i + 1], len = a.kv_len[i];
  w.slot = a.slots ? a.slots[i] : i;
  const bool ok = t0 >= 0 && t1 > t0 && t1 <= a.n_tok && len >= t1 - t0 && len <= (long long)a.max_pages * a.kv.page_size && w.slot >= 0 && w.slot < a.max_seqs;
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
      left -= tiles + AB_REST - skip;
      skip = 0;
      ++block;
      if (some) return true;
    }
  }
};

}  // namespace qie
