// rope_store.cu -- rotary positions of q and k and the store of k and v into the cache pages, one launch (qie_rope_rows, qie_rope_store).
//
//   (a, b) -> (a c - b s, b c + a s),  c, s = factor * cos, sin(pos * freq[i]),  in fp32 with one rounding
// The angle's turns pos * freq[i] / 2 pi are taken in 64 bits and only their fraction goes to 32: 2^31 positions leave it exact to 2^-20 of a turn.
//
// Bound by memory: every element is read and written once.  A CTA takes a few tokens: their cosines and sines go to shared memory (once a token, not once a
// head), then a thread takes the same place of the row in each token, V elements of a pair's first half and V of the second (or V / 2 neighbouring pairs),
// with the loads of four tokens under way.
#include <algorithm>

#include "common.cuh"
#include "kernels.h"
#include "launch.h"

namespace qie {
namespace {

constexpr int MOST_TOK = 8;  // tokens a CTA

template <int V>
struct Vec {
  uint32_t w[(V + 1) / 2];
};
template <int V>
__device__ __forceinline__ Vec<V> load(const bf16* p) {
  Vec<V> r;
  if constexpr (V == 8) {
    const uint4 t = *reinterpret_cast<const uint4*>(p);
    r.w[0] = t.x, r.w[1] = t.y, r.w[2] = t.z, r.w[3] = t.w;
  } else if constexpr (V == 4) {
    const uint2 t = *reinterpret_cast<const uint2*>(p);
    r.w[0] = t.x, r.w[1] = t.y;
  } else if constexpr (V == 2) {
    r.w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else {
    r.w[0] = *reinterpret_cast<const uint16_t*>(p);
  }
  return r;
}
template <int V>
__device__ __forceinline__ void store(bf16* p, const Vec<V>& r) {
  if constexpr (V == 8) *reinterpret_cast<uint4*>(p) = make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]);
  else if constexpr (V == 4) *reinterpret_cast<uint2*>(p) = make_uint2(r.w[0], r.w[1]);
  else if constexpr (V == 2) *reinterpret_cast<uint32_t*>(p) = r.w[0];
  else *reinterpret_cast<uint16_t*>(p) = (uint16_t)r.w[0];
}

// V elements at a time; NB: neighbours are pairs
template <int V, bool NB>
__global__ void rope_store_kernel(RopeArgs a, int n_tok) {
  constexpr bool SPLIT = !NB || V == 1;  // a pair's elements are loaded one by one
  extern __shared__ float2 cs[];  // [token][pair]
  __shared__ int s_pos[MOST_TOK];
  __shared__ long long s_at[MOST_TOK];  // offset of the token's cache row in the pool, below 0: none
  pdl_wait();
  pdl_trigger();
  const int t0 = blockIdx.x * n_tok, n = min(n_tok, a.n_tok - t0), hd = a.kv.hd, half = a.rotated / 2;
  for (int i = threadIdx.x; i < n * half; i += blockDim.x) {
    const int t = i / half;
    const double turns = (double)a.pos[t0 + t] * a.freq[i - t * half] * 0.15915494309189533577;
    float s, c;
    sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
    cs[i] = make_float2(c * a.factor, s * a.factor);
  }
  if (threadIdx.x < n) {
    const int t = threadIdx.x;
    s_pos[t] = a.pos[t0 + t];
    s_at[t] = -1;
    if (a.k) {
      const int row = a.row[t0 + t];
      if (row >= 0 && row < a.kv.n_pages * a.kv.page_size) s_at[t] = (long long)((size_t)(row / a.kv.page_size) * a.kv.page_stride() + (size_t)(row % a.kv.page_size) * hd);
    }
  }
  __syncthreads();
  // places of a row: of each head of q and k the pairs, then what is not turned; the heads of v
  const int other = NB ? 1 : half, pairs = SPLIT ? half / V : a.rotated / V, rest = (hd - a.rotated) / V, per = pairs + rest, n_kv = a.k ? a.kv.n_kv : 0;
  const int turned = (a.n_q + n_kv) * per, all = turned + n_kv * (hd / V);
  for (int u = threadIdx.x; u < all; u += blockDim.x) {
    int head, place, kind;  // 0: q, 1: k, 2: v
    if (u < turned) {
      head = u / per, place = u - head * per;
      kind = head >= a.n_q;
      if (kind) head -= a.n_q;
    } else {
      head = (u - turned) / (hd / V), place = u - turned - head * (hd / V);
      kind = 2;
    }
    const bool turn = kind < 2 && place < pairs;
    const int at = turn ? place * (NB && SPLIT ? 2 : V) : kind == 2 ? place * V : a.rotated + (place - pairs) * V;
    const size_t stride = kind == 0 ? a.q_stride : kind == 1 ? a.k_stride : a.v_stride;
    const bf16* src = (kind == 0 ? a.q : kind == 1 ? a.k : a.v) + (size_t)t0 * stride + (size_t)head * hd + at;
    bf16* dst = kind == 0 ? a.q_out + (size_t)t0 * a.q_out_stride + (size_t)head * hd + at : a.kv.chunk(0, a.layer, kind - 1, head) + at;
    constexpr int U = 4;
    for (int b = 0; b < n; b += U) {
      Vec<V> x[U], y[U];
#pragma unroll
      for (int e = 0; e < U; ++e)
        if (b + e < n) {
          x[e] = load<V>(src + (size_t)(b + e) * stride);
          if (SPLIT && turn) y[e] = load<V>(src + (size_t)(b + e) * stride + other);
        }
#pragma unroll
      for (int e = 0; e < U; ++e) {
        const int t = b + e;
        if (t >= n || (kind == 0 ? s_pos[t] < 0 : s_at[t] < 0)) continue;
        bf16* to = dst + (kind == 0 ? (size_t)t * a.q_out_stride : (size_t)s_at[t]);
        if (turn) {
          if constexpr (!SPLIT) {
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
              const float2 c = cs[t * half + place * (V / 2) + i];
              const float u0 = lo2f(x[e].w[i]), u1 = hi2f(x[e].w[i]);
              x[e].w[i] = pack2f(u0 * c.x - u1 * c.y, u1 * c.x + u0 * c.y);
            }
          } else if constexpr (V == 1) {
            const float2 c = cs[t * half + place];
            const float u0 = lo2f(x[e].w[0]), u1 = lo2f(y[e].w[0]);
            x[e].w[0] = pack2f(u0 * c.x - u1 * c.y, 0.f) & 0xffffu;
            y[e].w[0] = pack2f(u1 * c.x + u0 * c.y, 0.f) & 0xffffu;
          } else {
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
              const float2 c0 = cs[t * half + place * V + 2 * i], c1 = cs[t * half + place * V + 2 * i + 1];
              const float u0 = lo2f(x[e].w[i]), u1 = hi2f(x[e].w[i]), w0 = lo2f(y[e].w[i]), w1 = hi2f(y[e].w[i]);
              x[e].w[i] = pack2f(u0 * c0.x - w0 * c0.y, u1 * c1.x - w1 * c1.y);
              y[e].w[i] = pack2f(w0 * c0.x + u0 * c0.y, w1 * c1.x + u1 * c1.y);
            }
          }
          if constexpr (SPLIT) store<V>(to + other, y[e]);
        }
        store<V>(to, x[e]);
      }
    }
  }
}

template <int V, bool NB>
cudaError_t launch_v(const RopeArgs& a, cudaStream_t st) {
  const int hd = a.kv.hd, n_kv = a.k ? a.kv.n_kv : 0;
  const int per = (NB && V > 1 ? a.rotated : a.rotated / 2) / V + (hd - a.rotated) / V, all = (a.n_q + n_kv) * per + n_kv * (hd / V);
  int sms = 0, dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  sms = device_attribute<cudaDevAttrMultiProcessorCount>(dev);
  // as many tokens a CTA as leave four CTAs to an SM
  const int n_tok = std::max(1, std::min({MOST_TOK, a.n_tok / (4 * std::max(1, sms)), 4096 / a.rotated}));
  const int thr = std::min(256, (all + 31) / 32 * 32);
  return launched(launch_k(rope_store_kernel<V, NB>, dim3((a.n_tok + n_tok - 1) / n_tok), dim3(thr), n_tok * (a.rotated / 2) * sizeof(float2), st, a, n_tok));
}

}  // namespace

cudaError_t launch_rope_store(const RopeArgs& a, cudaStream_t st) {
  // the widest accesses that the head's parts, the rows' starts and their strides allow
  size_t all = (size_t)a.kv.hd | a.rotated | (a.neighbours ? 0 : a.rotated / 2);
  auto rows = [&](const void* p, size_t stride, int n) {
    if (p && n) all |= reinterpret_cast<uintptr_t>(p) / 2 | (a.n_tok > 1 ? stride : 0);
  };
  rows(a.q, a.q_stride, a.n_q), rows(a.q_out, a.q_out_stride, a.n_q);
  if (a.k) rows(a.k, a.k_stride, a.kv.n_kv), rows(a.v, a.v_stride, a.kv.n_kv), rows(a.kv.pool, 0, a.kv.n_kv);
  if (a.neighbours) return all % 8 == 0 ? launch_v<8, true>(a, st) : all % 4 == 0 ? launch_v<4, true>(a, st) : all % 2 == 0 ? launch_v<2, true>(a, st) : launch_v<1, true>(a, st);
  return all % 8 == 0 ? launch_v<8, false>(a, st) : all % 4 == 0 ? launch_v<4, false>(a, st) : all % 2 == 0 ? launch_v<2, false>(a, st) : launch_v<1, false>(a, st);
}

}  // namespace qie
