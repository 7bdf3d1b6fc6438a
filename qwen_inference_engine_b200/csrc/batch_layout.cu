// batch_layout.cu -- a step's layout on the device: from every request's cached and new tokens the rows of the step, their cache rows, the pages
// that the new tokens need and the pages that requests leave behind (qie_batch_layout).
//
//   n_i = max(new_i, 0), had_i = ceil(cached_i / P), need_i = ceil((cached_i + n_i) / P) - had_i, back_i = had_i where the request is over
//   token t of request i (t in [sum n_<i, sum n_<=i)): position p = cached_i + t - sum n_<i, its page the request's p / P -th:
//   the block table's where p / P < had_i, else ring[(first + sum need_<i + p / P - had_i) mod n_pages], which the table gets too
//
// Bound by latency: a launch, the requests' numbers, their sums, a page id a token.  Every CTA adds the requests up by itself (their numbers stay in shared memory), so none waits for
// another; a thread takes four tokens with one search.  B200, in a graph: 64 tokens of 64 requests 4.5 us, 8192 tokens of 340 requests 6.0, 131072 tokens of 1300 requests
// with 100 thousand pages given back 7.9.
#include <algorithm>

#include "cluster.cuh"
#include "common.cuh"
#include "kernels.h"
#include "launch.h"

namespace qie {
namespace {

constexpr int MOST_THR = 1024, MOST_CTA = 8, MOST_GRID = 256;

struct Sums {
  long long tok, need, back;
};
__device__ __forceinline__ Sums add(Sums a, Sums b) { return {a.tok + b.tok, a.need + b.need, a.back + b.back}; }
__device__ __forceinline__ Sums from_below(Sums v, int d) {
  return {__shfl_up_sync(0xffffffffu, v.tok, d), __shfl_up_sync(0xffffffffu, v.need, d), __shfl_up_sync(0xffffffffu, v.back, d)};
}

// what the CTA keeps of each request in shared memory: running sums of tokens, pages needed and pages given back, positions, row of the block table
struct Kept {
  int *tok, *need, *back, *cached, *slot;
  __device__ Kept(int* p, int n) : tok(p), need(p + n + 1), back(p + 2 * (n + 1)), cached(p + 3 * (n + 1)), slot(p + 4 * (n + 1)) {}
};
struct Request {
  int n, slot, cached, flags;
  Sums s;
};
__device__ __forceinline__ Request request(const BatchArgs& a, int i) {
  Request r{a.n_new[i], a.slots ? a.slots[i] : i, a.cached[i], 0, {0, 0, 0}};
  if (r.cached < 0 || r.n < -1 || r.slot < 0 || r.slot >= a.max_seqs) {
    r.flags = 8;
  } else if ((long long)r.cached + max(r.n, 0) > a.max_pages * a.page_size) {
    r.flags = 2;
  } else {
    const int had = (r.cached + a.page_size - 1) / a.page_size;
    r.s.tok = max(r.n, 0);
    r.s.need = r.n > 0 ? (r.cached + r.n + a.page_size - 1) / a.page_size - had : 0;
    r.s.back = r.n < 0 ? had : 0;
  }
  return r;
}
// the request that holds element x of the running sums s[0 .. n]: the last i with s[i] <= x (x < s[n])
__device__ __forceinline__ int holder(const int* s, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (s[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// n_tok_cta: CTAs that go through the tokens; those behind them, if there are, through the pages given back
__global__ void __launch_bounds__(MOST_THR) batch_layout_kernel(BatchArgs a, int wide, int cluster, int n_tok_cta) {
  extern __shared__ int kept_s[];
  __shared__ Sums warp_sums[MOST_THR / 32];
  __shared__ int flags_s;
  const Kept kept(kept_s, a.n_req);
  const int tid = threadIdx.x, thr = blockDim.x, lane = tid & 31, warp = tid >> 5;
  const int all = n_tok_cta * thr, me = blockIdx.x * thr + tid;  // of the tokens' threads
  const bool apart = gridDim.x > (unsigned)n_tok_cta;
  const int back_all = apart ? (gridDim.x - n_tok_cta) * thr : all, back_me = apart ? me - all : me;
  pdl_wait();
  pdl_trigger();
  if (tid == 0) flags_s = 0;
  const int first = a.ring_in[0], count = a.ring_in[1];
  // ---- running sums over the requests, a stretch of them a thread; every CTA for itself
  const int per = (a.n_req + thr - 1) / thr, i0 = min(a.n_req, tid * per), i1 = min(a.n_req, i0 + per);
  Sums mine{0, 0, 0};
  int flags = 0;
  Request one{};
  for (int i = i0; i < i1; ++i) {
    one = request(a, i);
    mine = add(mine, one.s);
    flags |= one.flags;
  }
  Sums run = mine;
  for (int d = 1; d < 32; d <<= 1) {
    const Sums o = from_below(run, d);
    if (lane >= d) run = add(run, o);
  }
  if (lane == 31) warp_sums[warp] = run;
  __syncthreads();
  if (flags) atomicOr(&flags_s, flags);
  Sums before{0, 0, 0}, total{0, 0, 0};
  for (int w = 0; w < thr / 32; ++w) {
    if (w == warp) before = total;
    total = add(total, warp_sums[w]);
  }
  Sums at{before.tok + run.tok - mine.tok, before.need + run.need - mine.need, before.back + run.back - mine.back};
  for (int i = i0; i < i1; ++i) {  // (a flag makes these sums useless, and nothing uses them)
    const Request r = per == 1 ? one : request(a, i);
    kept.tok[i] = (int)at.tok, kept.need[i] = (int)at.need, kept.back[i] = (int)at.back;
    kept.cached[i] = r.cached, kept.slot[i] = r.slot;
    if (blockIdx.x == 0) a.kv_len[i] = r.n < 0 ? 0 : r.cached + r.n, a.q_start[i] = (int)at.tok;
    at = add(at, r.s);
  }
  if (tid == 0) {
    kept.tok[a.n_req] = (int)total.tok, kept.need[a.n_req] = (int)total.need, kept.back[a.n_req] = (int)total.back;
    if (blockIdx.x == 0) a.q_start[a.n_req] = (int)total.tok;
  }
  __syncthreads();
  flags = flags_s;
  if (first < 0 || first >= a.n_pages || count < 0 || count > a.n_pages) flags |= 8;
  else if (total.need > count) flags |= 1;
  else if (count + total.back > a.n_pages) flags |= 8;
  if (total.tok > a.max_tokens) flags |= 4;
  const int n_tok = flags ? 0 : (int)total.tok, n_back = flags ? 0 : (int)total.back;
  if (flags && blockIdx.x == 0) {  // nothing to do for anybody
    for (int i = tid; i <= a.n_req; i += thr) a.q_start[i] = 0;
    for (int i = tid; i < a.n_req; i += thr) a.kv_len[i] = 0;
  }
  auto ring_at = [&](int i) {  // first + i modulo n_pages, i <= 2 n_pages
    long long x = (long long)first + i;
    while (x >= a.n_pages) x -= a.n_pages;
    return (int)x;
  };
  // ---- pages given back: behind the ring's last, so at none of the places that are read below
  for (int b = 4 * back_me; b >= 0 && b < n_back; b += 4 * back_all) {
    int i = holder(kept.back, a.n_req, b), page[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (b + e < n_back) {
        while (kept.back[i + 1] <= b + e) ++i;
        page[e] = a.block_table[(size_t)kept.slot[i] * a.max_pages + b + e - kept.back[i]];
      }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (b + e < n_back) a.free_ring[ring_at(count + b + e)] = page[e];
  }
  // ---- tokens, four a thread and step.  The one that begins a page takes it into the block table.
  for (int b = 4 * me; (int)blockIdx.x < n_tok_cta && b < a.max_tokens; b += 4 * all) {
    int pos[4], slot[4], row[4];
    int i = -1, end = 0, from = -1, page = 0;  // the request and its end; the first position of the page at hand
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int t = b + e;
      pos[e] = slot[e] = row[e] = -1;
      if (t >= n_tok) continue;
      if (t >= end) {
        i = e == 0 ? holder(kept.tok, a.n_req, t) : i + 1;
        while (kept.tok[i + 1] <= t) ++i;
        end = kept.tok[i + 1], from = -1;
      }
      const int p = kept.cached[i] + t - kept.tok[i];
      slot[e] = kept.slot[i];
      if (from < 0 || p - from >= a.page_size) {
        const int pg = p / a.page_size, had = (kept.cached[i] + a.page_size - 1) / a.page_size;
        int* at = a.block_table + (size_t)slot[e] * a.max_pages + pg;
        from = pg * a.page_size;
        page = pg < had ? *at : a.free_ring[ring_at(kept.need[i] + pg - had)];
        if (pg >= had && p == from) *at = page;
      }
      pos[e] = p;
      row[e] = (int)((unsigned)page * a.page_size + (unsigned)(p - from));
    }
    if (wide && b + 4 <= a.max_tokens) {
      *reinterpret_cast<int4*>(a.pos + b) = make_int4(pos[0], pos[1], pos[2], pos[3]);
      *reinterpret_cast<int4*>(a.slot + b) = make_int4(slot[0], slot[1], slot[2], slot[3]);
      *reinterpret_cast<int4*>(a.row + b) = make_int4(row[0], row[1], row[2], row[3]);
    } else {
      for (int e = 0; e < 4 && b + e < a.max_tokens; ++e) a.pos[b + e] = pos[e], a.slot[b + e] = slot[e], a.row[b + e] = row[e];
    }
  }
  // ---- the ring's state, which may be the word that the others read
  if (cluster) cluster_sync_all();
  if (me == 0) {
    a.status[0] = flags;
    a.status[1] = flags & 1 ? (int)min(total.need - count, 0x7fffffffll) : 0;
    a.ring_out[0] = flags ? first : ring_at((int)total.need);
    a.ring_out[1] = flags ? count : count - (int)total.need + n_back;
  }
}

}  // namespace

cudaError_t launch_batch_layout(const BatchArgs& a, cudaStream_t st) {
  static PerDeviceOnce set;
  if (set.need()) {
    const cudaError_t e = cudaFuncSetAttribute(batch_layout_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 5 * (BATCH_MAX_REQ + 1) * (int)sizeof(int));
    if (e != cudaSuccess) return e;
    set.done();
  }
  // A thread for four tokens and for a request.  Where the ring's state is updated in place the CTAs are one cluster (of eight at most): none may write it before all have
  // read it.  More than a few thousand tokens: half of the CTAs for the pages given back, which else come ahead of the tokens (8192 tokens, 2600 pages given back: 7.5 us,
  // so 6.0).  CTAs have 512 threads (with 1024 that case takes 8.4) but where a cluster of them is not enough (131072 tokens in place: 36 us, so 27; with a ring of its
  // own behind the step 7.9).
  const bool in_place = a.ring_in == a.ring_out || a.ring_in + 1 == a.ring_out || a.ring_in == a.ring_out + 1;
  const int quads = (a.max_tokens + 3) / 4, few = in_place && quads > MOST_CTA * 512 ? MOST_THR : 512;
  const int thr = std::min(few, std::max(128, (std::max(quads, a.n_req) + 31) / 32 * 32)), want = (quads + thr - 1) / thr;
  const int n_tok_cta = want > 1 ? std::min(want, (in_place ? MOST_CTA : MOST_GRID) / 2) : 1, ctas = want > 1 ? 2 * n_tok_cta : 1;
  const bool wide = ((reinterpret_cast<uintptr_t>(a.pos) | reinterpret_cast<uintptr_t>(a.slot) | reinterpret_cast<uintptr_t>(a.row)) & 15) == 0;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(thr);
  cfg.dynamicSmemBytes = 5 * (a.n_req + 1) * sizeof(int);
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  int na = 0;
  if (in_place && ctas > 1) {
    at[na].id = cudaLaunchAttributeClusterDimension;
    at[na].val.clusterDim.x = ctas;
    at[na].val.clusterDim.y = at[na].val.clusterDim.z = 1;
    ++na;
  }
  if (g_use_pdl) {
    at[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[na].val.programmaticStreamSerializationAllowed = 1;
    ++na;
  }
  cfg.attrs = at;
  cfg.numAttrs = na;
  return launched(cudaLaunchKernelEx(&cfg, batch_layout_kernel, a, (int)wide, (int)(in_place && ctas > 1), n_tok_cta));
}

}  // namespace qie
