// attn_batch.cu -- attention of a step's rows over the paged cache: requests with any number of rows, causal behind their cached positions, with an
// optional window (qie_attention_batch).
//
//   out_t = sum_j 2^(s (q_t . k_j) - m) v_j / sum_j 2^(s (q_t . k_j) - m) over the positions j that row t sees, m their running maximum
#include "common.cuh"
#include "kernels.h"
#include "launch.h"

namespace qie {
namespace {

// a warp a row and query head, one pass over the keys
template <int HD>
__global__ void __launch_bounds__(256) attn_batch_kernel(BatchAttnArgs a) {
  constexpr int E = HD / 32;
  pdl_wait();
  pdl_trigger();
  const int t = blockIdx.x, h = blockIdx.y * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (h >= a.n_q) return;
  // the request that owns the row
  int lo = 0, hi = a.n_req;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.q_start[mid] <= t) lo = mid;
    else hi = mid;
  }
  const int t0 = a.q_start[lo], t1 = a.q_start[lo + 1], slot = a.slots ? a.slots[lo] : lo;
  if (t < t0 || t >= t1 || slot < 0 || slot >= a.max_seqs) return;
  const long long most = (long long)a.max_pages * a.kv.page_size;
  const int len = (int)min((long long)max(a.kv_len[lo], 0), most), pos = min(len - 1, max(len - (t1 - t0), 0) + t - t0);
  const int kvh = h / (a.n_q / a.kv.n_kv);
  const int* bt = a.block_table + (size_t)slot * a.max_pages;
  float q[E], o[E], m = -INFINITY, l = 0.f;
  const bf16* src = a.q + t * a.q_stride + (size_t)h * HD + lane * E;
  for (int e = 0; e < E; ++e) q[e] = bf2f(src[e]), o[e] = 0.f;
  for (int j = a.window > 0 ? max(0, pos - a.window + 1) : 0; j <= pos; ++j) {
    const int page = bt[j / a.kv.page_size], at = j % a.kv.page_size;
    if (page < 0 || page >= a.kv.n_pages) continue;
    const bf16 *k = a.kv.chunk(page, a.layer, 0, kvh) + (size_t)at * HD + lane * E, *v = a.kv.chunk(page, a.layer, 1, kvh) + (size_t)at * HD + lane * E;
    float s = 0.f;
    for (int e = 0; e < E; ++e) s += q[e] * bf2f(k[e]);
    s = warp_sum(s) * a.scale_log2;
    const float top = fmaxf(m, s), f = exp2f(m - top), p = exp2f(s - top);
    l = l * f + p, m = top;
    for (int e = 0; e < E; ++e) o[e] = o[e] * f + p * bf2f(v[e]);
  }
  bf16* dst = a.out + t * a.out_stride + (size_t)h * HD + lane * E;
  for (int e = 0; e < E; ++e) dst[e] = f2bf(o[e] / l);
}

}  // namespace

size_t attention_batch_work(int, int) { return 16; }

cudaError_t launch_attention_batch(const BatchAttnArgs& a, cudaStream_t st) {
  const dim3 grid(a.n_tok, (a.n_q + 7) / 8);
  return launched(a.kv.hd == 64 ? launch_k(attn_batch_kernel<64>, grid, dim3(256), 0, st, a) : launch_k(attn_batch_kernel<128>, grid, dim3(256), 0, st, a));
}

}  // namespace qie
