// attn_batch_split.cuh -- what the kernels that share out a step's attention by attn_batch_plan.cuh have in common: a CTA's stretch, and the parts of items that
// were cut, joined by a second kernel.
#pragma once
#include "attn_batch_plan.cuh"
#include "common.cuh"
#include "launch.h"
#include "pack.cuh"
#include "tc_ptx.cuh"

namespace qie {

// sum over the block of a 64-bit value a thread: what the threads below have, and all
template <int NTHR>
__device__ __forceinline__ long long block_scan(long long v, long long* warp_sums, long long& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long run = v;
  for (int d = 1; d < 32; d <<= 1) {
    const long long o = __shfl_up_sync(0xffffffffu, run, d);
    if (lane >= d) run += o;
  }
  if (lane == 31) warp_sums[warp] = run;
  __syncthreads();
  long long before = 0;
  total = 0;
  for (int w = 0; w < NTHR / 32; ++w) {
    if (w == warp) before = total;
    total += warp_sums[w];
  }
  return before + run - v;
}

// a / b of numbers that are not below 0, mostly of 32 bits
__device__ __forceinline__ long long quotient(long long a, long long b) { return (a | b) >> 32 ? a / b : (long long)((unsigned)a / (unsigned)b); }

// What each CTA of a grid does: all costs of the step over the CTAs, and where in the requests its share begins (*s_walk, whose `left` is 0 before the call; in shared memory, there for the
// others behind the next barrier).
struct Stretch {
  long long share, x1;  // every CTA's, and this one's end
};
template <int NTHR>
__device__ __forceinline__ Stretch find_stretch(const BatchAttnArgs& a, int tt, long long* s_sums, Walk* s_walk) {
  const int tid = threadIdx.x, lane = tid & 31;
  const int per = (a.n_req + NTHR - 1) / NTHR, r0 = min(a.n_req, tid * per), r1 = min(a.n_req, r0 + per);
  long long mine = 0, total, head = 0;  // head: a kv head's cost of the thread's last request
  for (int i = r0; i < r1; ++i) {
    const Raw w = request(a, i, tt);
    head = ab_cost(w.r, w.r.nb, tt, a.window, ab_rest(a));
    mine += a.kv.n_kv * head;
  }
  const long long below = block_scan<NTHR>(mine, s_sums, total);
  const long long share = quotient(total + gridDim.x - 1, gridDim.x), x0 = min(total, share * blockIdx.x), x1 = min(total, x0 + share);
  const bool own = x0 < x1 && below <= x0 && x0 < below + mine;
  if (const unsigned owner = __ballot_sync(0xffffffffu, own)) {  // the warp of the thread that has the request in which it begins
    int req = 0;
    long long rest = 0;
    if (own) {
      rest = x0 - below;
      for (req = r0; req < r1 - 1; ++req) {
        const Raw w = request(a, req, tt);
        const long long h = ab_cost(w.r, w.r.nb, tt, a.window, ab_rest(a));
        if (rest < a.kv.n_kv * h) {
          head = h;
          break;
        }
        rest -= a.kv.n_kv * h;
      }
    }
    const int from = __ffs(owner) - 1;
    req = __shfl_sync(0xffffffffu, req, from), rest = __shfl_sync(0xffffffffu, rest, from), head = __shfl_sync(0xffffffffu, head, from);
    const Raw w = request(a, req, tt);
    const int kvh = (int)quotient(rest, head);
    rest -= kvh * head;
    // the block in which it begins: the last one whose cost of blocks before is not above the rest, 32 at a time
    int lo = 0, hi = w.r.nb;
    long long before = 0;
    while (hi - lo > 1) {
      const int step = (hi - lo + 31) / 32, x = lo + lane * step;
      const long long c = x < hi ? ab_cost(w.r, x, tt, a.window, ab_rest(a)) : rest + 1;
      const int k = 31 - __clz(__ballot_sync(0xffffffffu, c <= rest));  // (lane 0's is)
      before = __shfl_sync(0xffffffffu, c, k);
      hi = min(hi, lo + (k + 1) * step), lo += k * step;
    }
    if (lane == 0) *s_walk = Walk{w, req, kvh, lo, (int)(rest - before), x1 - x0};
  }
  return Stretch{share, x1};
}

// The work area: of each CTA what there is to join of the item that begins there and goes on behind it; then two parts of each CTA, of the item that began before it and of
// the one that goes on: O, four columns of all rows after four columns of all rows, so that threads with rows side by side write and read side by side, maxima, sums.
struct JoinInfo {
  int t0, tokens, kvh, parts;  // rows t0 .. t0 + tokens of Q; parts 0: nothing
};
template <int HD, int ROWS>
constexpr int PART = ROWS * HD + 2 * ROWS;  // floats


// The parts of an item that was cut into the rows of its result: CTA k joins the item that CTA k of the kernel above began and did not end.  Sums are taken in a fixed
// order.
constexpr int JOIN_THR = 512;
// 2^(m - top): a row sees nothing of some parts, and a sum that is no number counts whatever the maximum beside it
__device__ __forceinline__ float weight(float m, float l, float top) { return l != l ? l : m > -INFINITY ? ex2_tc(m - top) : 0.f; }
struct Sum4 {
  float m = -INFINITY, l = 0.f;
  float4 o = {0.f, 0.f, 0.f, 0.f};
  __device__ __forceinline__ void add(float pm, float pl, const float4& x) {
    const float top = fmaxf(m, pm), f = weight(m, l, top), pf = weight(pm, pl, top);
    m = top;
    l = l * f + pl * pf;
    o.x *= f, o.y *= f, o.z *= f, o.w *= f;
    if (pf != 0.f) o.x += x.x * pf, o.y += x.y * pf, o.z += x.z * pf, o.w += x.w * pf;
  }
};
// ROWS of a part; a block's rows are `g` query heads of a token, or, where a group has more, `subs` blocks share it (their kv heads are counted on: kv head * subs + block)
struct JoinShape {
  int g, group, subs;
};
template <int HD, int ROWS>
__device__ __forceinline__ void join_parts(const BatchAttnArgs& a, const JoinShape& sh, int n_cta, int of, int part_of_rows, Sum4* sums) {  // of: the CTA of the kernel above; of many rows' columns the part
  constexpr int C = HD / 4;  // groups of columns
  constexpr bool MANY = ROWS * C > JOIN_THR;  // rows enough for more than one step of a CTA's threads
  const JoinInfo* info = reinterpret_cast<const JoinInfo*>(a.work);
  JoinInfo in = info[of];
  int slice = part_of_rows, cta = of, slices = 1;  // of many rows' columns; of few rows' columns, where an item has many parts: the CTAs behind the first have none that begin there
  if constexpr (!MANY) {
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const JoinInfo x = info[max(of - s, 0)];
      const int share = x.parts >= 5 ? 4 : x.parts >= 3 ? 2 : 1;
      if (x.parts > 1 && s < share && s <= of) in = x, slice = s, cta = of - s, slices = share;
    }
  }
  const float* first = reinterpret_cast<const float*>(info + n_cta) + ((size_t)cta * 2 + 1) * PART<HD, ROWS>;
  const int sub = sh.subs > 1 ? in.kvh % sh.subs : 0, G = min(sh.g, sh.group - sub * sh.g), head0 = (sh.subs > 1 ? in.kvh / sh.subs : in.kvh) * sh.group + sub * sh.g;
  const int rows = in.tokens * G, n = in.parts, tid = threadIdx.x;
  // (a work area that two calls used at once must not lead outside)
  if (n <= 1 || n > n_cta - cta || rows <= 0 || rows > ROWS || in.t0 < 0 || in.t0 > a.n_tok - in.tokens || in.kvh < 0 || in.kvh >= a.kv.n_kv * sh.subs) return;
  bf16* out = a.out + (size_t)in.t0 * a.out_stride + (size_t)head0 * HD;
  auto store = [&](int row, int c, const float4& o, float f) {
    *reinterpret_cast<uint2*>(out + (size_t)(row / G) * a.out_stride + (size_t)(row % G) * HD + c * 4) = make_uint2(pack2f(o.x * f, o.y * f), pack2f(o.z * f, o.w * f));
  };
  auto part_of = [&](int q) { return first + (q == 0 ? 0 : (size_t)(2 * q - 1) * PART<HD, ROWS>); };  // the others are the first ones of the CTAs behind
  const int all = rows * C;
  if (MANY && all > JOIN_THR) {
    // many rows: four threads a row with every fourth group of its columns; a part's weight is the row's
    constexpr int MINE = C / (JOIN_THR / ROWS) > 0 ? C / (JOIN_THR / ROWS) : 1;
    const int row = tid % ROWS, c0 = tid / ROWS;
    if (row >= rows) return;
    float top = -INFINITY, sum = 0.f;
    for (int q = 0; q < n; q += 4) {
      float m[4], l[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float* part = part_of(min(q + u, n - 1)) + ROWS * HD + row;
        m[u] = q + u < n ? part[0] : -INFINITY, l[u] = q + u < n ? part[ROWS] : 0.f;
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float t = fmaxf(top, m[u]);
        sum = sum * weight(top, sum, t) + l[u] * weight(m[u], l[u], t);
        top = t;
      }
    }
    const float inv = sum > 0.f ? 1.f / sum : sum;
#pragma unroll 1
    for (int b = 4 * slice; b < min(MINE, 4 * slice + 4); b += 4) {
      float4 o[4] = {};
#pragma unroll 2
      for (int q = 0; q < n; ++q) {
        const float* part = part_of(q);
        float4 x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = *reinterpret_cast<const float4*>(part + ((c0 + (b + e) * (JOIN_THR / ROWS)) * ROWS + row) * 4);
        const float f = weight(part[ROWS * HD + row], part[ROWS * HD + ROWS + row], top) * inv;
        if (f != 0.f)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e].x += x[e].x * f, o[e].y += x[e].y * f, o[e].z += x[e].z * f, o[e].w += x[e].w * f;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) store(row, c0 + (b + e) * (JOIN_THR / ROWS), o[e], 1.f);
    }
    return;
  }
  if (MANY && slice) return;
  // few rows: four columns of a row a thread, and the parts in turn with the threads that are left
  constexpr int U = 4;
  const int mine = all / slices, lanes = JOIN_THR / mine, i = tid % mine, q0 = tid / mine, c = i / rows + slice * (C / slices) * !MANY, row = i % rows;
  Sum4 s;
  if (q0 < lanes)
    for (int q = q0; q < n; q += U * lanes) {
      float m[U], l[U];
      float4 x[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int k = q + u * lanes;
        m[u] = -INFINITY, l[u] = 0.f;
        if (k >= n) continue;
        const float* part = part_of(k);
        m[u] = part[ROWS * HD + row], l[u] = part[ROWS * HD + ROWS + row];
        x[u] = *reinterpret_cast<const float4*>(part + (c * ROWS + row) * 4);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (q + u * lanes < n) s.add(m[u], l[u], x[u]);
    }
  sums[tid] = s;
  __syncthreads();
  if (q0 == 0) {
    for (int w = 1; w < min(lanes, n); ++w) s.add(sums[w * mine + i].m, sums[w * mine + i].l, sums[w * mine + i].o);
    store(row, c, s.o, s.l > 0.f ? 1.f / s.l : s.l);
  }
}


template <int HD, int ROWS>
__global__ void __launch_bounds__(JOIN_THR, 2) attn_batch_join_kernel(BatchAttnArgs a, JoinShape sh, int n_cta) {
  __shared__ Sum4 sums[JOIN_THR];
  pdl_wait();
  pdl_trigger();
  join_parts<HD, ROWS>(a, sh, n_cta, blockIdx.x, blockIdx.y, sums);
}
template <int HD, int ROWS>
inline cudaError_t launch_join(const BatchAttnArgs& a, const JoinShape& sh, int ctas, cudaStream_t st) {
  constexpr int SLICES = ROWS * (HD / 4) > JOIN_THR ? HD / 4 / (JOIN_THR / ROWS) / 4 : 1;
  return launched(launch_k(attn_batch_join_kernel<HD, ROWS>, dim3(ctas, SLICES), dim3(JOIN_THR), 0, st, a, sh, ctas));
}

}  // namespace qie
