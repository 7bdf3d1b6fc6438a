// batch_layout.cu -- a step's layout on the device: from every request's cached and new tokens the rows of the step, their cache rows, the pages
// that the new tokens need and the pages that requests leave behind (qie_batch_layout).
//
//   n_i = max(new_i, 0), had_i = ceil(cached_i / P), need_i = ceil((cached_i + n_i) / P) - had_i, back_i = had_i where the request is over
//   token t of request i (t in [sum n_<i, sum n_<=i)): position p = cached_i + t - sum n_<i, its page the request's p / P -th:
//   the block table's where p / P < had_i, else ring[(first + sum need_<i + p / P - had_i) mod n_pages], which the table gets too
#include "common.cuh"
#include "kernels.h"
#include "launch.h"

namespace qie {
namespace {

constexpr int NTHR = 1024;

struct Sums {
  long long tok, need, back;
};
__device__ __forceinline__ Sums add(Sums a, Sums b) { return {a.tok + b.tok, a.need + b.need, a.back + b.back}; }
__device__ __forceinline__ Sums from_below(Sums v, int d) {
  return {__shfl_up_sync(0xffffffffu, v.tok, d), __shfl_up_sync(0xffffffffu, v.need, d), __shfl_up_sync(0xffffffffu, v.back, d)};
}

struct Request {
  int tok, need, back, had, flags;
};
__device__ __forceinline__ Request request(const BatchArgs& a, int i) {
  const int c = a.cached[i], n = a.n_new[i], slot = a.slots ? a.slots[i] : i;
  Request r{0, 0, 0, 0, 0};
  if (c < 0 || n < -1 || slot < 0 || slot >= a.max_seqs) {
    r.flags = 8;
  } else if ((long long)c + max(n, 0) > (long long)a.max_pages * a.page_size) {
    r.flags = 2;
  } else {
    r.had = (int)(((long long)c + a.page_size - 1) / a.page_size);
    r.tok = max(n, 0);
    r.need = n > 0 ? (int)(((long long)c + n + a.page_size - 1) / a.page_size) - r.had : 0;
    r.back = n < 0 ? r.had : 0;
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

__global__ void __launch_bounds__(NTHR) batch_layout_kernel(BatchArgs a) {
  extern __shared__ int sums[];
  __shared__ Sums warp_sums[NTHR / 32];
  __shared__ int flags_s;
  int *tok = sums, *need = tok + a.n_req + 1, *back = need + a.n_req + 1;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_wait();
  pdl_trigger();
  if (tid == 0) flags_s = 0;
  const int first = a.ring_in[0], count = a.ring_in[1];
  __syncthreads();
  // ---- running sums over the requests, a stretch of them a thread
  const int per = (a.n_req + NTHR - 1) / NTHR, i0 = min(a.n_req, tid * per), i1 = min(a.n_req, i0 + per);
  Sums mine{0, 0, 0};
  int flags = 0;
  for (int i = i0; i < i1; ++i) {
    const Request r = request(a, i);
    mine = add(mine, Sums{r.tok, r.need, r.back});
    flags |= r.flags;
  }
  Sums run = mine;
  for (int d = 1; d < 32; d <<= 1) {
    const Sums o = from_below(run, d);
    if (lane >= d) run = add(run, o);
  }
  if (lane == 31) warp_sums[warp] = run;
  if (flags) atomicOr(&flags_s, flags);
  __syncthreads();
  Sums before{0, 0, 0}, total{0, 0, 0};
  for (int w = 0; w < NTHR / 32; ++w) {
    if (w == warp) before = total;
    total = add(total, warp_sums[w]);
  }
  flags = flags_s;
  if (first < 0 || first >= a.n_pages || count < 0 || count > a.n_pages) flags |= 8;
  else if (total.need > count) flags |= 1;
  else if (count + total.back > a.n_pages) flags |= 8;
  if (total.tok > a.max_tokens) flags |= 4;
  if (tid == 0) {
    a.status[0] = flags;
    a.status[1] = flags & 1 ? (int)min(total.need - count, 0x7fffffffll) : 0;
  }
  if (flags) {  // nothing to do for anybody
    for (int i = tid; i <= a.n_req; i += NTHR) a.q_start[i] = 0;
    for (int i = tid; i < a.n_req; i += NTHR) a.kv_len[i] = 0;
    for (int t = tid; t < a.max_tokens; t += NTHR) a.pos[t] = a.slot[t] = a.row[t] = -1;
    if (tid == 0) a.ring_out[0] = first, a.ring_out[1] = count;
    return;
  }
  Sums at{before.tok + run.tok - mine.tok, before.need + run.need - mine.need, before.back + run.back - mine.back};
  for (int i = i0; i < i1; ++i) {
    const Request r = request(a, i);
    tok[i] = (int)at.tok, need[i] = (int)at.need, back[i] = (int)at.back;
    a.q_start[i] = (int)at.tok;
    a.kv_len[i] = a.n_new[i] < 0 ? 0 : a.cached[i] + r.tok;
    at = add(at, Sums{r.tok, r.need, r.back});
  }
  if (tid == 0) {
    tok[a.n_req] = (int)total.tok, need[a.n_req] = (int)total.need, back[a.n_req] = (int)total.back;
    a.q_start[a.n_req] = (int)total.tok;
  }
  __syncthreads();
  // ---- pages taken and given back.  The places written in the ring are behind its last page, so none that is read.
  auto ring_at = [&](int i) { return (int)(((long long)first + i) % a.n_pages); };
  auto row_of = [&](int i) { return a.block_table + (size_t)(a.slots ? a.slots[i] : i) * a.max_pages; };
  auto had_of = [&](int i) { return (int)(((long long)a.cached[i] + a.page_size - 1) / a.page_size); };
  for (int j = tid; j < (int)total.need; j += NTHR) {
    const int i = holder(need, a.n_req, j);
    row_of(i)[had_of(i) + j - need[i]] = a.free_ring[ring_at(j)];
  }
  for (int j = tid; j < (int)total.back; j += NTHR) {
    const int i = holder(back, a.n_req, j);
    a.free_ring[ring_at(count + j)] = row_of(i)[j - back[i]];
  }
  // ---- tokens
  for (int t = tid; t < a.max_tokens; t += NTHR) {
    int pos = -1, slot = -1, row = -1;
    if (t < (int)total.tok) {
      const int i = holder(tok, a.n_req, t);
      pos = a.cached[i] + t - tok[i];
      slot = a.slots ? a.slots[i] : i;
      const int had = had_of(i), pg = pos / a.page_size;
      const int page = pg < had ? row_of(i)[pg] : a.free_ring[ring_at(need[i] + pg - had)];
      row = page * a.page_size + pos - pg * a.page_size;
    }
    a.pos[t] = pos, a.slot[t] = slot, a.row[t] = row;
  }
  if (tid == 0) a.ring_out[0] = ring_at((int)total.need), a.ring_out[1] = count - (int)total.need + (int)total.back;
}

}  // namespace

cudaError_t launch_batch_layout(const BatchArgs& a, cudaStream_t st) {
  static PerDeviceOnce set;
  if (set.need()) {
    const cudaError_t e = cudaFuncSetAttribute(batch_layout_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 3 * (BATCH_MAX_REQ + 1) * (int)sizeof(int));
    if (e != cudaSuccess) return e;
    set.done();
  }
  return launched(launch_k(batch_layout_kernel, dim3(1), dim3(NTHR), 3 * (a.n_req + 1) * sizeof(int), st, a));
}

}  // namespace qie
