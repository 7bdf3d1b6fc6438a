// attn_batch_plan_check.cpp -- how csrc/attn_batch.cu shares out a step (csrc/attn_batch_plan.cuh) against counting one by one, on the host.  Arguments: seed, steps.
// Prints "ok" and what was counted, or the line of the first check that does not hold.
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <map>
#include <random>
#include <tuple>
#include <vector>

#include "attn_batch_plan.cuh"

using namespace qie;

#define CHECK(x)                                       \
  do {                                                 \
    if (!(x)) {                                        \
      printf("line %d: %s\n", __LINE__, #x);           \
      return false;                                    \
    }                                                  \
  } while (0)

static std::mt19937 rng;
static int upto(int n) { return (int)(rng() % (unsigned)n); }

// costs of the first blocks of one request, by a sum over the blocks, and the tiles of a block by its positions
static bool costs(long& counted) {
  const int tt = 1 + upto(128), kind = upto(5);
  AbRequest r;
  r.n = 1 + upto(kind == 0 ? 1 : kind == 1 ? 5 : kind == 2 ? 200 : 6000);
  r.c = upto(3) == 0 ? 0 : upto(7) == 0 ? (1 << 30) - r.n - upto(1000) : upto(50000);
  r.nb = (r.n + tt - 1) / tt;
  const int window = upto(2) ? 0 : upto(9) == 0 ? 2147483647 : 1 + upto(upto(2) ? 100 : 60000);
  long long sum = 0;
  for (int b = 0; b < r.nb; ++b) {
    CHECK(ab_cost(r, b, tt, window) == sum);
    int first, last;
    ab_tiles(r, b, tt, window, first, last);
    const long long p0 = (long long)r.c + (long long)b * tt, p1 = std::min((long long)r.c + r.n, p0 + tt) - 1, low = window ? std::max(0ll, p0 - window + 1) : 0;
    CHECK(first == low / AB_TK && last == p1 / AB_TK + 1);
    sum += last - first + AB_REST;
    ++counted;
  }
  CHECK(ab_cost(r, r.nb, tt, window) == sum);
  return true;
}

struct Part {
  int begin, end, tiles, cta;
};
// a step's pieces: every tile of every item once, in its order, by CTAs side by side; the parts of an item where the kernel that joins them looks for them
static bool step(long& pieces, long& cut) {
  const int kind = upto(4), n_req = kind == 0 ? 1 : 1 + upto(kind == 1 ? 300 : 20), nkv = 1 + upto(4);
  const bool few = upto(3) == 0, bad_offsets = upto(11) == 0;
  const int G = 1 + upto(few ? 16 : 128), tt = (few ? 16 : AB_TQ) / G, ctas = upto(4) ? 296 : 1 + upto(400);
  std::vector<int> start(n_req + 1), len(n_req), slot(n_req);
  for (int i = 0; i < n_req; ++i) {
    const int n = upto(4) == 0 ? 0 : upto(2) ? 1 : 1 + upto(upto(3) ? 30 : 900);
    start[i + 1] = start[i] + n, len[i] = n + (upto(3) ? upto(3000) : 0), slot[i] = i;
    if (upto(50) == 0) len[i] = n - 1;
    if (upto(50) == 0) slot[i] = -3;
  }
  BatchAttnArgs a{};
  a.n_tok = start[n_req];
  if (bad_offsets)
    for (int& s : start)
      if (upto(5) == 0) s = (int)rng();
  a.q_start = start.data(), a.kv_len = len.data(), a.slots = slot.data();
  a.n_req = n_req, a.max_seqs = n_req, a.max_pages = 1000, a.n_q = G * nkv, a.window = upto(2) ? 0 : 1 + upto(500);
  a.kv.n_kv = nkv, a.kv.page_size = 16;

  std::vector<long long> below(n_req + 1);
  size_t items_wanted = 0;
  for (int i = 0; i < n_req; ++i) {
    const Raw w = request(a, i, tt);
    below[i + 1] = below[i] + nkv * ab_cost(w.r, w.r.nb, tt, a.window);
    items_wanted += (size_t)w.r.nb * nkv;
  }
  const long long total = below[n_req], share = (total + ctas - 1) / ctas;
  std::map<std::tuple<int, int, int>, std::vector<Part>> items;  // {first row, kv head, its position}
  std::map<int, std::pair<std::tuple<int, int, int>, int>> begun;  // by the CTA: the item that goes on behind it, and its parts
  for (int k = 0; k < ctas; ++k) {
    const long long x0 = std::min(total, share * k), x1 = std::min(total, x0 + share);
    if (x0 >= x1) continue;
    const int req = (int)(std::upper_bound(below.begin(), below.end(), x0) - below.begin()) - 1;
    const Raw w = request(a, req, tt);
    const long long head = ab_cost(w.r, w.r.nb, tt, a.window), rest = (x0 - below[req]) % head;
    // the search of a warp for the block in which the CTA begins
    int lo = 0, hi = w.r.nb;
    while (hi - lo > 1) {
      const int by = (hi - lo + 31) / 32;
      unsigned in = 0;
      for (int lane = 0; lane < 32; ++lane)
        if (lo + lane * by < hi && ab_cost(w.r, lo + lane * by, tt, a.window) <= rest) in |= 1u << lane;
      CHECK(in & 1);
      const int at = 31 - __builtin_clz(in);
      CHECK(in == (at == 31 ? ~0u : (2u << at) - 1));
      hi = std::min(hi, lo + (at + 1) * by), lo += at * by;
    }
    Walk walk{w, req, (int)((x0 - below[req]) / head), lo, (int)(rest - ab_cost(w.r, lo, tt, a.window)), x1 - x0};
    CHECK(walk.kvh < nkv && walk.skip >= 0);
    Piece p;
    for (bool first = true; walk.next(a, tt, p); first = false) {
      ++pieces;
      CHECK(p.begin < p.end && p.end <= p.tiles && (first || p.begin == 0) && p.tokens >= 1 && p.tokens <= tt && p.kvh >= 0 && p.kvh < nkv);
      CHECK(p.t0 >= 0 && p.t0 + p.tokens <= a.n_tok && p.limit <= 1000 * 16 && p.pos0 + p.tokens <= p.limit);
      const int low0 = a.window ? std::max(0, p.pos0 - a.window + 1) : 0, low1 = a.window ? std::max(0, p.pos0 + p.tokens - a.window) : 0, end = p.key0 + p.tiles * AB_TK;
      CHECK(p.key0 <= low0 && p.key0 + AB_TK > low0 && end - AB_TK <= p.pos0 + p.tokens - 1 && end > p.pos0 + p.tokens - 1);
      int edges = 0;
      for (int i = p.begin; i < p.end; ++i) edges += p.key0 + i * AB_TK + AB_TK > p.pos0 + 1 || p.key0 + i * AB_TK < low1;
      CHECK(edges <= (few ? 4 : 6));
      const std::tuple<int, int, int> item{p.t0, p.kvh, p.pos0};
      items[item].push_back({p.begin, p.end, p.tiles, k});
      if (!p.whole() && p.begin == 0) begun[k] = {item, (int)((x1 - p.left + p.tiles - 1) / share) - k + 1};
    }
  }
  if (bad_offsets) return true;  // (items may share rows)
  CHECK(items.size() == items_wanted);
  for (const auto& [item, parts] : items) {
    int at = 0;
    for (size_t j = 0; j < parts.size(); ++j) {
      CHECK(parts[j].begin == at && (j == 0 || parts[j].cta == parts[j - 1].cta + 1));
      at = parts[j].end;
    }
    CHECK(at == parts[0].tiles);
    if (parts.size() == 1) continue;
    ++cut;
    const auto b = begun.find(parts[0].cta);
    CHECK(b != begun.end() && b->second.first == item && b->second.second == (int)parts.size());
  }
  return true;
}

// the largest call: a block a token
static bool largest() {
  AbRequest r{(1 << 24) - 1, 5, (1 << 24) - 1};
  long long sum = 0;
  for (int b = 0; b < r.nb; ++b) {
    int first, last;
    ab_tiles(r, b, 1, 0, first, last);
    sum += last - first + AB_REST;
  }
  CHECK(sum == ab_cost(r, r.nb, 1, 0));
  return true;
}

int main(int, char** argv) {
  rng.seed((unsigned)atoi(argv[1]));
  long counted = 0, pieces = 0, cut = 0;
  for (int i = 0; i < 10 * atoi(argv[2]); ++i)
    if (!costs(counted)) return 1;
  for (int i = 0; i < atoi(argv[2]); ++i)
    if (!step(pieces, cut)) return 1;
  if (!largest()) return 1;
  printf("ok: %ld blocks, %ld pieces, %ld items that are cut\n", counted, pieces, cut);
}
