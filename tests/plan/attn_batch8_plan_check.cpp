// attn_batch8_plan_check.cpp -- how csrc/attn_batch8.cu shares out a step over its two kernels (csrc/attn_batch_plan.cuh): each token of each kv head in one item of one of them, each tile of an
// item once, parts where the kernel that joins looks for them.  On the host.  Arguments: seed, steps.
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <map>
#include <random>
#include <tuple>
#include <vector>

#include "attn_batch_plan.cuh"

using namespace qie;

#define CHECK(x)                             \
  do {                                       \
    if (!(x)) {                              \
      printf("line %d: %s\n", __LINE__, #x); \
      return false;                          \
    }                                        \
  } while (0)

static std::mt19937 rng;
static int upto(int n) { return (int)(rng() % (unsigned)n); }

struct Part {
  int begin, end, tiles, cta;
};
// one kernel's pieces; `seen`: of a token and head how many items have it
static bool plan(const BatchAttnArgs& a, int tt, int ctas, std::vector<int>& seen, long& pieces, long& cut) {
  const int rest_of = ab_rest(a);
  std::vector<long long> below(a.n_req + 1);
  for (int i = 0; i < a.n_req; ++i) {
    const Raw w = request(a, i, tt);
    below[i + 1] = below[i] + a.kv.n_kv * ab_cost(w.r, w.r.nb, tt, a.window, rest_of);
  }
  const long long total = below[a.n_req], share = (total + ctas - 1) / ctas;
  std::map<std::tuple<int, int>, std::vector<Part>> items;  // {first row, kv head}
  std::map<int, std::pair<std::tuple<int, int>, int>> begun;
  for (int k = 0; k < ctas; ++k) {
    const long long x0 = std::min(total, share * k), x1 = std::min(total, x0 + share);
    if (x0 >= x1) continue;
    const int req = (int)(std::upper_bound(below.begin(), below.end(), x0) - below.begin()) - 1;
    const Raw w = request(a, req, tt);
    const long long head = ab_cost(w.r, w.r.nb, tt, a.window, rest_of), rest = (x0 - below[req]) % head;
    int block = 0;
    while (block + 1 < w.r.nb && ab_cost(w.r, block + 1, tt, a.window, rest_of) <= rest) ++block;
    Walk walk{w, req, (int)((x0 - below[req]) / head), block, (int)(rest - ab_cost(w.r, block, tt, a.window, rest_of)), x1 - x0};
    Piece p;
    for (bool first = true; walk.next(a, tt, p); first = false) {
      ++pieces;
      CHECK(p.begin < p.end && p.end <= p.tiles && (first || p.begin == 0) && p.tokens >= 1 && p.tokens <= tt && p.kvh >= 0 && p.kvh < a.kv.n_kv && p.t0 >= 0 && p.t0 + p.tokens <= a.n_tok);
      const std::tuple<int, int> item{p.t0, p.kvh};
      if (p.begin == 0)
        for (int t = p.t0; t < p.t0 + p.tokens; ++t) ++seen[(size_t)t * a.kv.n_kv + p.kvh];
      items[item].push_back({p.begin, p.end, p.tiles, k});
      if (!p.whole() && p.begin == 0) begun[k] = {item, (int)((x1 - p.left + p.tiles - 1) / share) - k + 1};
    }
  }
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

static bool step(long& pieces, long& cut) {
  const int n_req = 1 + upto(upto(2) ? 200 : 12), nkv = 1 + upto(4), group = 1 + upto(upto(3) ? 16 : 128), hd = upto(2) ? 64 : 128, g = std::min(group, 16), subs = (group + g - 1) / g;
  const int kind = upto(4);  // 0: single rows
  std::vector<int> start(n_req + 1), len(n_req);
  for (int i = 0; i < n_req; ++i) {
    const int n = upto(5) == 0 ? 0 : kind == 0 || upto(2) ? 1 : 1 + upto(upto(2) ? 40 : 900);
    start[i + 1] = start[i] + n, len[i] = n + (upto(3) ? upto(3000) : 0);
    if (upto(50) == 0) len[i] = n - 1;
  }
  BatchAttnArgs a{};
  a.n_tok = start[n_req] + upto(9), a.q_start = start.data(), a.kv_len = len.data();
  a.n_req = n_req, a.max_seqs = n_req, a.max_pages = 1000, a.n_q = group * nkv, a.window = upto(2) ? 0 : 1 + upto(500);
  a.kv.n_kv = nkv, a.kv.page_size = 16;
  BatchAttnArgs small = a, large = a;
  small.kv.n_kv *= subs, small.rest = 7, large.rest = hd == 64 ? 5 : 8;
  const bool few = a.n_tok <= a.n_req;
  std::vector<int> in_small((size_t)a.n_tok * small.kv.n_kv), in_large((size_t)a.n_tok * nkv);
  if (!few) {
    small.n_most = large.n_more = 16 / g;
    if (!plan(large, 256 / group, 148, in_large, pieces, cut)) return false;
  }
  if (!plan(small, (group <= 8 ? 8 : 16) / g, 296, in_small, pieces, cut)) return false;
  std::vector<int> wanted(a.n_tok);
  for (int i = 0; i < n_req; ++i)
    for (int t = start[i]; t < start[i + 1]; ++t) wanted[t] = len[i] >= start[i + 1] - start[i];
  for (int t = 0; t < a.n_tok; ++t)
    for (int h = 0; h < nkv; ++h) {
      int blocks = 0;
      for (int s = 0; s < subs; ++s) {
        const int x = in_small[((size_t)t * nkv + h) * subs + s];
        CHECK(x == 0 || x == 1);
        blocks += x;
      }
      CHECK(blocks == 0 || blocks == subs);
      CHECK((blocks == subs) + in_large[(size_t)t * nkv + h] == wanted[t]);
    }
  return true;
}

int main(int, char** argv) {
  rng.seed((unsigned)atoi(argv[1]));
  long pieces = 0, cut = 0;
  for (int i = 0; i < atoi(argv[2]); ++i)
    if (!step(pieces, cut)) return 1;
  printf("ok: %ld pieces, %ld items that are cut\n", pieces, cut);
}
