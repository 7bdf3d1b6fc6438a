// rope_store.cu -- rotary positions of q and k and the store of k and v into the cache pages, one launch (qie_rope_rows, qie_rope_store).
//
//   (a, b) -> (a c - b s, b c + a s),  c, s = factor * cos, sin(pos * freq[i]),  in fp32 with one rounding
// The angle's turns pos * freq[i] / 2 pi are taken in 64 bits and only their fraction goes to 32: 2^31 positions leave it exact to 2^-20 of a turn.
#include "common.cuh"
#include "kernels.h"
#include "launch.h"

namespace qie {
namespace {

constexpr int NTHR = 256;

// one CTA a token
__global__ void __launch_bounds__(NTHR) rope_store_kernel(RopeArgs a) {
  extern __shared__ float2 cs[];  // of the token's pairs
  pdl_wait();
  pdl_trigger();
  const int t = blockIdx.x, pos = a.pos[t], hd = a.kv.hd, half = a.rotated / 2;
  const long long row = a.k ? a.row[t] : -1;
  const bool put = row >= 0 && row < (long long)a.kv.n_pages * a.kv.page_size;
  for (int i = threadIdx.x; i < half; i += NTHR) {
    const double turns = (double)pos * a.freq[i] * 0.15915494309189533577;
    float s, c;
    sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
    cs[i] = make_float2(c * a.factor, s * a.factor);
  }
  __syncthreads();
  auto turn = [&](const bf16* x, bf16* y) {  // a head
    for (int i = threadIdx.x; i < half; i += NTHR) {
      const int ia = a.neighbours ? 2 * i : i, ib = a.neighbours ? 2 * i + 1 : i + half;
      const float u = bf2f(x[ia]), w = bf2f(x[ib]);
      y[ia] = f2bf(u * cs[i].x - w * cs[i].y);
      y[ib] = f2bf(w * cs[i].x + u * cs[i].y);
    }
    for (int i = a.rotated + threadIdx.x; i < hd; i += NTHR) y[i] = x[i];
  };
  if (pos >= 0)
    for (int h = 0; h < a.n_q; ++h) turn(a.q + t * a.q_stride + (size_t)h * hd, a.q_out + t * a.q_out_stride + (size_t)h * hd);
  if (put) {
    const int page = (int)(row / a.kv.page_size), at = (int)(row % a.kv.page_size);
    for (int h = 0; h < a.kv.n_kv; ++h) {
      turn(a.k + t * a.k_stride + (size_t)h * hd, a.kv.chunk(page, a.layer, 0, h) + (size_t)at * hd);
      for (int i = threadIdx.x; i < hd; i += NTHR) (a.kv.chunk(page, a.layer, 1, h) + (size_t)at * hd)[i] = a.v[t * a.v_stride + (size_t)h * hd + i];
    }
  }
}

}  // namespace

cudaError_t launch_rope_store(const RopeArgs& a, cudaStream_t st) {
  return launched(launch_k(rope_store_kernel, dim3(a.n_tok), dim3(NTHR), a.rotated / 2 * sizeof(float2), st, a));
}

}  // namespace qie
