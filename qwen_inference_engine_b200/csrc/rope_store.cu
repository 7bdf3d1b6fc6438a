// rope_store.cu -- rotary positions of q and k and the store of k and v into the cache pages, one launch (qie_rope_rows, qie_rope_store).
//
//   (a, b) -> (a c - b s, b c + a s),  c, s = factor * cos, sin(pos * freq[i]),  in fp32 with one rounding
// A pair's turns a position, freq[i] / 2 pi, are kept as their fraction in 64-bit fixed point (of the nearest double); their product with the position modulo 2^64 is the
// fraction of the turns at that position, off by at most 2^31 times half a unit of the double: 2^-23 of a turn.  Sine and cosine of that, in [-pi, pi], by the hardware's
// functions: 2^-20.5 of one, where results are rounded to 2^-8 of themselves.  (In doubles, with the library's functions, the angles were a third of the kernel's
// instructions.)
//
// Bound by memory: every element is read and written once.  A thread has one place of the row (V elements of a pair's first half and V of the second, or V / 2
// neighbouring pairs) and goes through groups of U tokens: the next group's loads are under way while it turns the one at hand, and the CTA's threads compute the next
// group's cosines and sines, once a token, into the other half of shared memory.
// B200, in a graph with inputs that are not in L2: 8192 tokens of 12 + 2 x 2 heads of 128, 67 MB, 15.5 us (a copy of as many bytes 12.8); 20011 tokens of 14 + 2 x 2 heads of
// 64, half of each turned, 92 MB, 21.7; 64 tokens 2.6.
#include <algorithm>

#include "common.cuh"
#include "kernels.h"
#include "launch.h"

namespace qie {
namespace {

constexpr int MOST_THR = 512;

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

// two fp32 values at once
struct Two {
  unsigned long long v;
  __device__ __forceinline__ Two(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
  __device__ __forceinline__ explicit Two(uint32_t w) : Two(lo2f(w), hi2f(w)) {}
  __device__ __forceinline__ uint32_t rounded() const {
    float a, b;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
    return pack2f(a, b);
  }
};
__device__ __forceinline__ Two operator*(Two a, Two b) {
  asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(a.v) : "l"(b.v));
  return a;
}
__device__ __forceinline__ Two operator-(Two a, Two b) {
  asm("sub.rn.f32x2 %0, %0, %1;" : "+l"(a.v) : "l"(b.v));
  return a;
}
__device__ __forceinline__ Two fma(Two a, Two b, Two c) {
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(c.v) : "l"(a.v), "l"(b.v));
  return c;
}

// V elements at a time; NB: neighbours are pairs
template <int V, bool NB, int U>
__global__ void __launch_bounds__(MOST_THR, 2) rope_store_kernel(RopeArgs a) {
  constexpr bool SPLIT = !NB || V == 1;  // a pair's elements are loaded one by one
  constexpr int EACH = SPLIT ? V : V / 2;  // pairs of a place
  constexpr int W = EACH > 1 ? 2 : 1;  // pairs together: their cosines, then their sines
  extern __shared__ __align__(16) float cs[];  // [2][token][W pairs of the place][place]: threads at places side by side read side by side; then the pairs' turns
  // of the groups at hand, next and behind that: positions, and offsets of the tokens' cache rows in the pool (below 0: none)
  __shared__ int s_pos[4][U];
  __shared__ long long s_at[4][U];
  pdl_wait();
  pdl_trigger();
  const int hd = a.kv.hd, half = a.rotated / 2, tid = threadIdx.x, thr = blockDim.x;
  unsigned long long* turns_s = reinterpret_cast<unsigned long long*>(cs + (2 * U * a.rotated + 1) / 2 * 2);
  for (int p = tid; p < half; p += thr) {
    const double turns = a.freq[p] * 0.15915494309189533577;
    turns_s[p] = (unsigned long long)((turns - floor(turns)) * 18446744073709551616.0);
  }
  // places of a row: of each head of q and k the pairs, then what is not turned; the heads of v
  const int other = NB ? 1 : half, pairs = half / EACH, rest = (hd - a.rotated) / V, per = pairs + rest, n_kv = a.k ? a.kv.n_kv : 0;
  const int turned = (a.n_q + n_kv) * per, all = turned + n_kv * (hd / V), u = blockIdx.y * thr + tid;
  int place = 0, kind = -1;  // 0: q, 1: k, 2: v, below 0: none
  bool turn = false;
  size_t stride = 0;
  const bf16* src = nullptr;
  bf16* dst = nullptr;
  if (u < all) {
    int head;
    if (u < turned) {
      head = u / per, place = u - head * per;
      kind = head >= a.n_q;
      if (kind) head -= a.n_q;
    } else {
      head = (u - turned) / (hd / V), place = u - turned - head * (hd / V);
      kind = 2;
    }
    turn = kind < 2 && place < pairs;
    const int at = turn ? place * (NB && SPLIT ? 2 : V) : kind == 2 ? place * V : a.rotated + (place - pairs) * V;
    stride = kind == 0 ? a.q_stride : kind == 1 ? a.k_stride : a.v_stride;
    src = (kind == 0 ? a.q : kind == 1 ? a.k : a.v) + (size_t)head * hd + at;
    dst = kind == 0 ? a.q_out + (size_t)head * hd + at : a.kv.chunk(0, a.layer, kind - 1, head) + at;
  }
  struct Group {
    Vec<V> x[U], y[U];
  };
  auto fetch = [&](int t0, Group& g) {
#pragma unroll
    for (int e = 0; e < U; ++e)
      if (kind >= 0 && t0 + e < a.n_tok) {
        const bf16* from = src + (size_t)(t0 + e) * stride;
        g.x[e] = load<V>(from);
        if (SPLIT && turn) g.y[e] = load<V>(from + other);
      }
  };
  const int dt = thr / half, dp = thr - dt * half;
  auto angles = [&](int t0, int k) {  // of the k-th group, whose positions are there
    const int n = min(U, a.n_tok - t0);
    float* c = cs + (k & 1) * U * a.rotated;
    for (int t = tid / half, p = tid - t * half; t < n;) {
      const int j = p % EACH;
      const int turns = (int)((unsigned long long)(unsigned)s_pos[k & 3][t] * turns_s[p] >> 32);  // their fraction, in 2^-32 of a turn from -1/2 on
      float sn, cn;
      __sincosf((float)turns * 1.4629180792671596e-9f, &sn, &cn);  // (2 pi / 2^32)
      float* at = c + t * a.rotated + ((j / W) * pairs + p / EACH) * 2 * W + j % W;
      at[0] = cn * a.factor, at[W] = sn * a.factor;
      t += dt, p += dp;
      if (p >= half) p -= half, ++t;
    }
  };
  int pos = -1, row = -1;
  auto ask = [&](int t0) {  // a token's numbers, one of the first threads each
    if (tid < U && t0 + tid < a.n_tok) pos = a.pos[t0 + tid], row = a.k ? a.row[t0 + tid] : -1;
  };
  auto note = [&](int k) {
    if (tid >= U) return;
    s_pos[k & 3][tid] = pos;
    s_at[k & 3][tid] = row >= 0 && row < a.kv.n_pages * a.kv.page_size
                           ? (long long)((size_t)(row / a.kv.page_size) * a.kv.page_stride() + (size_t)(row % a.kv.page_size) * hd) : -1;
  };
  auto put = [&](int t0, int k, Group& g) {
    if (kind < 0) return;
#pragma unroll
    for (int e = 0; e < U; ++e) {
      if (t0 + e >= a.n_tok) break;
      const long long at = s_at[k & 3][e];
      if (kind == 0 ? s_pos[k & 3][e] < 0 : at < 0) continue;
      bf16* to = dst + (kind == 0 ? (size_t)(t0 + e) * a.q_out_stride : (size_t)at);
      Vec<V> &x = g.x[e], &y = g.y[e];
      if (turn) {
        const float* mine = cs + ((k & 1) * U + e) * a.rotated + place * 2 * W;
        if constexpr (!SPLIT && W == 2) {
#pragma unroll
          for (int i = 0; i < V / 2; i += 2) {
            const float4 f = *reinterpret_cast<const float4*>(mine + i * pairs * 2);
            const float u0 = lo2f(x.w[i]), u1 = hi2f(x.w[i]), u2 = lo2f(x.w[i + 1]), u3 = hi2f(x.w[i + 1]);
            x.w[i] = pack2f(u0 * f.x - u1 * f.z, u1 * f.x + u0 * f.z);
            x.w[i + 1] = pack2f(u2 * f.y - u3 * f.w, u3 * f.y + u2 * f.w);
          }
        } else if constexpr (!SPLIT) {
          const float u0 = lo2f(x.w[0]), u1 = hi2f(x.w[0]);
          x.w[0] = pack2f(u0 * mine[0] - u1 * mine[1], u1 * mine[0] + u0 * mine[1]);
        } else if constexpr (V == 1) {
          const float u0 = lo2f(x.w[0]), u1 = lo2f(y.w[0]);
          x.w[0] = pack2f(u0 * mine[0] - u1 * mine[1], 0.f) & 0xffffu;
          y.w[0] = pack2f(u1 * mine[0] + u0 * mine[1], 0.f) & 0xffffu;
        } else {
#pragma unroll
          for (int i = 0; i < V / 2; ++i) {
            const float4 f = *reinterpret_cast<const float4*>(mine + i * pairs * 4);
            const Two c(f.x, f.y), s(f.z, f.w), v(x.w[i]), w(y.w[i]);
            x.w[i] = (v * c - w * s).rounded();
            y.w[i] = fma(v, s, w * c).rounded();
          }
        }
        if constexpr (SPLIT) store<V>(to + other, y);
      }
      store<V>(to, x);
    }
  };
  const int step = gridDim.x * U;
  Group g;
  int t = blockIdx.x * U, k = 0;
  ask(t);
  fetch(t, g);
  note(0);
  ask(t + step);
  __syncthreads();
  angles(t, 0);
  note(1);
  for (;; ++k) {
    __syncthreads();
    const int next = t + step;
    if (next >= a.n_tok) break;
    Group h;
    ask(next + step);
    fetch(next, h);
    put(t, k, g);
    angles(next, k + 1);
    note(k + 2);
    g = h;
    t = next;
  }
  put(t, k, g);
}

template <int V, bool NB>
cudaError_t launch_v(const RopeArgs& a, cudaStream_t st) {
  constexpr int EACH = NB && V > 1 ? V / 2 : V;
  const int hd = a.kv.hd, n_kv = a.k ? a.kv.n_kv : 0;
  const int per = a.rotated / 2 / EACH + (hd - a.rotated) / V, all = (a.n_q + n_kv) * per + n_kv * (hd / V);
  int dev = 0;
  const cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const int sms = std::max(1, device_attribute<cudaDevAttrMultiProcessorCount>(dev));
  // A thread a place; CTAs that an SM has room for at once (at 64 registers a thread) go through the tokens.  Groups are of two tokens where a place has two loads, else of four
  // (20011 tokens by twos 23.8 us, by fours 21.7; 8192 tokens with two loads by fours 18.8, by twos 15.5); of one where the tokens are too few for all SMs (64 tokens).
  constexpr int U = NB ? 4 : 2;
  const int ny = (all + MOST_THR - 1) / MOST_THR, thr = ((all + ny - 1) / ny + 31) / 32 * 32, most = std::max(1, 1024 / thr) * sms;
  const int groups = (a.n_tok + U - 1) / U;
  auto bytes = [&](int u) { return ((2 * u * a.rotated + 1) / 2 * 2 + a.rotated) * sizeof(float); };
  if ((long long)groups * ny >= 2 * sms)
    return launched(launch_k(rope_store_kernel<V, NB, U>, dim3(std::max(1, std::min(groups, most / ny)), ny), dim3(thr), bytes(U), st, a));
  return launched(launch_k(rope_store_kernel<V, NB, 1>, dim3(a.n_tok, ny), dim3(thr), bytes(1), st, a));
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
