// kv8_store.cu -- rotary positions of q and k and the store of k and v into a cache of 8 bits, one launch (qie_rope_store8), and its rows read back (qie_kv8_read).
//
// Positions as in rope_store.cu: turns in 64-bit fixed point.  Keys are turned in fp32 and coded from there, without a rounding to bf16 between; so that few of them come to the other side
// of a border between two codes, cosines and sines are rounded from 64 bits (with the hardware's functions, 2^-20.5, the codes' error beside the exact rotation's was twice that of a rotation
// in fp32 from exact cosines).
// A warp takes a token and some of its heads, eight elements a lane, so that a head is 8 or 16 lanes: cosines and sines are computed once for all of them, a lane's share each, a pair's other
// half is a shuffle away, and so is the largest element.  Queries are loaded four groups at a time (two 16.5 us and three 15.9 for the first call below with the hardware's cosines, four 16.6; for
// the second 25.9, 26.3 and 24.5), the first groups before the token's position and row are there; four CTAs an SM (three 17.3 and 24.6, five, of fewer registers, 20.7 and 28.6).
// Every element is read and written once.  B200, in a graph: 8192 tokens of 12 + 2 x 2 heads of 128, 63 MB, 17.0 us (3.7 TB/s; the store of bf16 keys and values 15.5: a wave and a half of
// CTAs, and the shuffles and conversions of their instructions); 20011 of 14 + 2 x 2 of 64 in int8, half of each rotated, stored and read back 26.7; 64 of 28 + 2 x 4 of 128 3.0, a launch.
#include <algorithm>

#include "common.cuh"
#include "kernels.h"
#include "kv8.cuh"
#include "launch.h"

namespace qie {
namespace {

constexpr int THR = 256, WARPS = THR / 32;
enum { TURN_NONE, TURN_NEIGHBOURS, TURN_LANES, TURN_ANY };  // pairs: none; within a lane; of lanes half / 8 apart; of any elements

// Division by the page size: floor(n / P) = n * m >> (31 + s) for n < 2^31, s = ceil(log2 P), m = ceil(2^(31 + s) / P) (what m has too much, n times it, is below 2^31 * P / 2^(31 + s) <= 1
// of a unit of the quotient's fraction of 1 / P).
struct PageDiv {
  uint32_t m;
  int shift;
  explicit PageDiv(int P) {
    int s = 0;
    while ((1ll << s) < P) ++s;
    shift = 31 + s;
    m = (uint32_t)(((1ull << shift) + P - 1) / P);
  }
  __device__ __forceinline__ int operator()(int n) const { return (int)((unsigned long long)n * m >> shift); }
};
// a layer's vector of head 0 in cache row `row`: its key; its value is n_kv * page_size vectors behind, the next head page_size
__device__ __forceinline__ size_t vec_of(const Kv8Geom& kv, const PageDiv& div, int layer, int row) {
  const int page = div(row);
  return ((size_t)page * kv.n_layers + layer) * 2 * kv.n_kv * kv.page_size + (row - page * kv.page_size);
}

// cosine and sine of t / 2^64 turns, times a factor
__device__ __forceinline__ float2 cos_sin(unsigned long long t, double factor) {
  double s, c;
  sincospi((double)(long long)t * (1.0 / 9223372036854775808.0), &s, &c);
  return make_float2((float)(c * factor), (float)(s * factor));
}

template <int HD, int CODE, int TURN, bool WIDE>
__global__ void __launch_bounds__(THR, 4) rope_store8_kernel(Rope8Args a, PageDiv div, int chunks, int per) {
  constexpr int LH = HD / 8, HW = 32 / LH;                                             // lanes of a head, heads of a warp at a time: a group
  constexpr int NP = TURN == TURN_NEIGHBOURS ? 4 : TURN == TURN_NONE ? 1 : 8, U = 4;  // pairs that the lane has a part of; groups ahead
  __shared__ uint4 s_row[TURN == TURN_ANY ? WARPS * HW * LH : 1];  // (a type with the alignment of its accesses)
  __shared__ unsigned long long s_turns[HD / 2];          // of the pairs a position, their fraction in 2^-64
  __shared__ __align__(16) float2 s_cs[WARPS][HD / 2];  // of a warp's token
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane / LH, p = lane % LH, e0 = p * 8;
  const int half = a.rotated / 2, n_kv = a.kv.n_kv;
  const int gq = (a.n_q + HW - 1) / HW, gk = (n_kv + HW - 1) / HW, groups = gq + 2 * gk;
  if (TURN != TURN_NONE) {
    for (int i = threadIdx.x; i < half; i += THR) {
      const double w = a.freq[i] * 0.15915494309189533577;
      s_turns[i] = (unsigned long long)((w - floor(w)) * 18446744073709551616.0);
    }
    __syncthreads();
  }
  const long long all = (long long)a.n_tok * chunks;
  for (long long w = (long long)blockIdx.x * WARPS + warp; w < all; w += (long long)gridDim.x * WARPS) {
    const int t = chunks == 1 ? (int)w : (int)(w / chunks), chunk = (int)(w - (long long)t * chunks);
    const int pos = TURN == TURN_NONE ? 0 : a.pos[t], row = a.row[t];
    const bool kept = row >= 0 && row < a.kv.n_pages * a.kv.page_size;
    const int g0 = chunk * per, g1 = min(groups, g0 + per);
    auto load = [&](const bf16* src, bool yes, uint32_t (&x)[4]) {
      if (!yes) {
        x[0] = x[1] = x[2] = x[3] = 0;
      } else if constexpr (WIDE) {
        const uint4 v = *reinterpret_cast<const uint4*>(src);
        x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = pack2(src[2 * j], src[2 * j + 1]);
      }
    };
    const bf16 *src_q = a.q + (size_t)t * a.q_stride + sub * HD + e0, *src_k = a.k + (size_t)t * a.k_stride + sub * HD + e0, *src_v = a.v + (size_t)t * a.v_stride + sub * HD + e0;
    // of the queries' groups U at a time, and the first of keys and values; these before the token's numbers are there
    const int q1 = min(g1, gq), k0 = max(g0 - gq, 0), k1 = min(g1 - gq, gk), v0 = max(g0 - gq - gk, 0), v1 = g1 - gq - gk;
    uint32_t x[U][4], xk[4], xv[4];
    auto fetch = [&](int g) {
#pragma unroll
      for (int u = 0; u < U; ++u) load(src_q + (g + u) * (HW * HD), g + u < q1 && (g + u) * HW + sub < a.n_q, x[u]);
    };
    fetch(g0);
    load(src_k + k0 * (HW * HD), k0 < k1 && k0 * HW + sub < n_kv, xk);
    load(src_v + v0 * (HW * HD), v0 < v1 && v0 * HW + sub < n_kv, xv);
    float c[NP], s[NP];
    if constexpr (TURN != TURN_NONE) {
      __syncwarp();
      for (int i = lane; i < half; i += 32) {
        s_cs[warp][i] = cos_sin((unsigned long long)(unsigned)pos * s_turns[i], a.factor);
      }
      __syncwarp();
      const bool on = e0 < a.rotated;
      const int first = !on ? 0 : TURN == TURN_NEIGHBOURS ? e0 / 2 : e0 < half ? e0 : e0 - half;
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        if constexpr (TURN == TURN_LANES) {  // (a multiple of eight pairs)
          if (j % 2 == 0) {
            const float4 f = *reinterpret_cast<const float4*>(&s_cs[warp][first + j]);
            c[j] = on ? f.x : 1.f, c[j + 1] = on ? f.z : 1.f;
            s[j] = !on ? 0.f : e0 < half ? -f.y : f.y, s[j + 1] = !on ? 0.f : e0 < half ? -f.w : f.w;
          }
        } else {
          const int e = TURN == TURN_NEIGHBOURS ? e0 + 2 * j : e0 + j, i = TURN == TURN_NEIGHBOURS ? e / 2 : e < half ? e : e - half;
          const float2 f = s_cs[warp][e < a.rotated ? i : 0];
          c[j] = e < a.rotated ? f.x : 1.f, s[j] = e >= a.rotated ? 0.f : TURN == TURN_ANY && e < half ? -f.y : f.y;
        }
      }
    }
    auto turn = [&](const uint32_t (&x)[4], float (&y)[8]) {  // (all lanes together)
      if constexpr (TURN == TURN_NEIGHBOURS) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float u = lo2f(x[j]), v = hi2f(x[j]);
          y[2 * j] = u * c[j] - v * s[j], y[2 * j + 1] = v * c[j] + u * s[j];
        }
      } else if constexpr (TURN == TURN_LANES) {
        const int d = half / 8, from = e0 < half ? lane + d : e0 < a.rotated ? lane - d : lane;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t o = __shfl_sync(0xffffffffu, x[j], from);
          y[2 * j] = lo2f(x[j]) * c[2 * j] + lo2f(o) * s[2 * j], y[2 * j + 1] = hi2f(x[j]) * c[2 * j + 1] + hi2f(o) * s[2 * j + 1];
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) y[2 * j] = lo2f(x[j]), y[2 * j + 1] = hi2f(x[j]);
        if constexpr (TURN == TURN_ANY) {
          uint4* head = s_row + (warp * HW + sub) * LH;
          const bf16* mine = reinterpret_cast<const bf16*>(head);
          __syncwarp();
          head[p] = make_uint4(x[0], x[1], x[2], x[3]);
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int e = e0 + j;
            if (e < a.rotated) y[j] = y[j] * c[j] + bf2f(mine[e < half ? e + half : e - half]) * s[j];
          }
        }
      }
    };
    bf16* dst = a.q_out + (size_t)t * a.q_out_stride + sub * HD + e0;
    for (int g = g0; g < q1;) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (g + u >= q1) break;
        float y[8];
        turn(x[u], y);
        if ((g + u) * HW + sub < a.n_q && pos >= 0) {
          bf16* to = dst + (g + u) * (HW * HD);
          if constexpr (WIDE) {
            *reinterpret_cast<uint4*>(to) = make_uint4(pack2f(y[0], y[1]), pack2f(y[2], y[3]), pack2f(y[4], y[5]), pack2f(y[6], y[7]));
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) to[j] = f2bf(y[j]);
          }
        }
      }
      g += U;
      if (g < q1) fetch(g);
    }
    if (!kept) continue;  // (the warp's: a token's cache row)
    const size_t vec0 = vec_of(a.kv, div, a.layer, row) + (size_t)sub * a.kv.page_size;
    auto code = [&](const float (&y)[8], int g, bool is_v) {
      uint32_t most = 0;  // of the bits without signs: infinities and what is no number are above all numbers
#pragma unroll
      for (int j = 0; j < 8; ++j) most = max(most, __float_as_uint(y[j]) & 0x7fffffffu);
#pragma unroll
      for (int d = 1; d < LH; d <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, d));
      if (g * HW + sub >= n_kv) return;
      const uint32_t byte = kv8_scale_byte<CODE>(most);
      const float f = kv8_inverse(byte);
      const size_t vec = vec0 + (size_t)(g * HW + (is_v ? n_kv : 0)) * a.kv.page_size;
      uint2 w = make_uint2(0, 0);
      if (byte != 255) w = make_uint2(kv8_pack<CODE>(y[0] * f, y[1] * f, y[2] * f, y[3] * f), kv8_pack<CODE>(y[4] * f, y[5] * f, y[6] * f, y[7] * f));
      *reinterpret_cast<uint2*>(a.kv.codes + vec * HD + e0) = w;
      if (p == 0) a.kv.scale[vec] = (uint8_t)byte;
    };
    for (int g = k0; g < k1; ++g) {
      float y[8];
      if (g > k0) load(src_k + g * (HW * HD), g * HW + sub < n_kv, xk);
      turn(xk, y);
      code(y, g, false);
    }
    for (int g = v0; g < v1; ++g) {
      float y[8];
      if (g > v0) load(src_v + g * (HW * HD), g * HW + sub < n_kv, xv);
#pragma unroll
      for (int j = 0; j < 4; ++j) y[2 * j] = lo2f(xv[j]), y[2 * j + 1] = hi2f(xv[j]);
      code(y, g, true);
    }
  }
}

template <int HD, int CODE, int TURN>
cudaError_t launch_turn(const Rope8Args& a, bool wide, cudaStream_t st) {
  constexpr int HW = 32 / (HD / 8);
  int dev = 0;
  const cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const int sms = std::max(1, device_attribute<cudaDevAttrMultiProcessorCount>(dev));
  // A token's heads are shared out over several warps where the tokens are too few to give every SM sixteen.
  const int groups = (a.n_q + HW - 1) / HW + 2 * ((a.kv.n_kv + HW - 1) / HW);
  const int want = std::min(groups, std::max(1, 16 * sms / a.n_tok)), per = (groups + want - 1) / want, chunks = (groups + per - 1) / per;
  const long long warps = (long long)a.n_tok * chunks;
  const int ctas = (int)std::min<long long>((warps + WARPS - 1) / WARPS, 8ll * sms);
  if (wide) return launched(launch_k(rope_store8_kernel<HD, CODE, TURN, true>, dim3(ctas), dim3(THR), 0, st, a, PageDiv(a.kv.page_size), chunks, per));
  return launched(launch_k(rope_store8_kernel<HD, CODE, TURN, false>, dim3(ctas), dim3(THR), 0, st, a, PageDiv(a.kv.page_size), chunks, per));
}
template <int HD, int CODE>
cudaError_t launch_code(const Rope8Args& a, bool wide, cudaStream_t st) {
  if (!a.freq) return launch_turn<HD, CODE, TURN_NONE>(a, wide, st);
  if (a.neighbours) return launch_turn<HD, CODE, TURN_NEIGHBOURS>(a, wide, st);
  return a.rotated % 16 == 0 ? launch_turn<HD, CODE, TURN_LANES>(a, wide, st) : launch_turn<HD, CODE, TURN_ANY>(a, wide, st);
}

// Sixteen elements a thread, which has one place of a row (k or v, head, piece) and goes through rows U at a time: their indexes, then scales and codes, then results.  Bound by memory: 32768
// rows of 4 x 2 heads of 128, 101 MB, 18.6 us, 5.4 TB/s; 701 of 2 x 2 of 64 1.7, a launch.  With a place a thread found by divisions, a row at a time, and results of 16 bytes 24.1.
template <int CODE, int W>  // W: elements of a result's access, 16, 8 or 1
__global__ void __launch_bounds__(THR) kv8_read_kernel(Kv8ReadArgs a, PageDiv div, int wide, int deep) {  // wide x deep threads: places of a row, rows
  constexpr int U = 4;
  pdl_wait();
  pdl_trigger();
  const int hd = a.kv.hd, pieces = hd / 16, half = a.kv.n_kv * pieces, place = blockIdx.y * wide + threadIdx.x % wide, lane_row = threadIdx.x / wide;
  if (place >= 2 * half || lane_row >= deep) return;
  const int is_v = place >= half, head = (place - is_v * half) / pieces, piece = (place - is_v * half) % pieces;
  bf16* dst = is_v ? a.v : a.k;
  if (!dst) return;
  dst += head * hd + piece * 16;
  const size_t stride = is_v ? a.v_stride : a.k_stride, off = (size_t)(is_v * a.kv.n_kv + head) * a.kv.page_size;
  const int step = gridDim.x * deep, end = a.kv.n_pages * a.kv.page_size;
  for (long long r0 = (long long)blockIdx.x * deep + lane_row; r0 < a.n_rows; r0 += (long long)U * step) {
    int row[U];
    uint32_t byte[U];
    uint4 code[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long r = r0 + (long long)u * step;
      row[u] = r < a.n_rows ? a.row[r] : -1;
      if (row[u] >= end) row[u] = -1;
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (row[u] >= 0) {
        const size_t vec = vec_of(a.kv, div, a.layer, row[u]) + off;
        byte[u] = a.kv.scale[vec];
        code[u] = *reinterpret_cast<const uint4*>(a.kv.codes + vec * hd + piece * 16);
      }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (row[u] >= 0) {
        const float f = kv8_scale(byte[u]);
        const uint32_t w[4] = {code[u].x, code[u].y, code[u].z, code[u].w};
        uint32_t o[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t lo, hi;
          kv8_unpack<CODE>(w[j], lo, hi);
          o[2 * j] = pack2f(h_lo(lo) * f, h_hi(lo) * f), o[2 * j + 1] = pack2f(h_lo(hi) * f, h_hi(hi) * f);
        }
        bf16* to = dst + (size_t)(r0 + (long long)u * step) * stride;
        if constexpr (W == 16) {
          asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(to), "r"(o[0]), "r"(o[1]), "r"(o[2]), "r"(o[3]), "r"(o[4]), "r"(o[5]), "r"(o[6]), "r"(o[7]) : "memory");
        } else if constexpr (W == 8) {
          *reinterpret_cast<uint4*>(to) = make_uint4(o[0], o[1], o[2], o[3]);
          *reinterpret_cast<uint4*>(to + 8) = make_uint4(o[4], o[5], o[6], o[7]);
        } else {
          uint16_t* t16 = reinterpret_cast<uint16_t*>(to);
#pragma unroll
          for (int j = 0; j < 8; ++j) t16[2 * j] = (uint16_t)o[j], t16[2 * j + 1] = (uint16_t)(o[j] >> 16);
        }
      }
  }
}

}  // namespace

cudaError_t launch_rope_store8(const Rope8Args& a, cudaStream_t st) {
  size_t all = 0;  // rows on 16-byte boundaries?
  auto rows = [&](const void* p, size_t stride) { all |= reinterpret_cast<uintptr_t>(p) / 2 | (a.n_tok > 1 ? stride : 0); };
  if (a.n_q) rows(a.q, a.q_stride), rows(a.q_out, a.q_out_stride);
  rows(a.k, a.k_stride), rows(a.v, a.v_stride);
  const bool wide = all % 8 == 0;
  if (a.kv.hd == 64) return a.kv.code == KV8_E4M3 ? launch_code<64, KV8_E4M3>(a, wide, st) : launch_code<64, KV8_INT8>(a, wide, st);
  return a.kv.code == KV8_E4M3 ? launch_code<128, KV8_E4M3>(a, wide, st) : launch_code<128, KV8_INT8>(a, wide, st);
}

cudaError_t launch_kv8_read(const Kv8ReadArgs& a, cudaStream_t st) {
  int dev = 0;
  const cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const int sms = std::max(1, device_attribute<cudaDevAttrMultiProcessorCount>(dev));
  size_t off = 0;
  auto rows = [&](const void* p, size_t stride) {
    if (p) off |= reinterpret_cast<uintptr_t>(p) / 2 | (a.n_rows > 1 ? stride : 0);
  };
  rows(a.k, a.k_stride), rows(a.v, a.v_stride);
  const int places = 2 * a.kv.n_kv * (a.kv.hd / 16), wide = std::min(places, THR), deep = THR / wide, ny = (places + wide - 1) / wide;
  const dim3 grid((unsigned)std::min<long long>(((long long)a.n_rows + deep - 1) / deep, std::max(1, 4 * sms / ny)), ny), block(THR);
  const PageDiv div(a.kv.page_size);
  auto go = [&](auto kernel) { return launched(launch_k(kernel, grid, block, 0, st, a, div, wide, deep)); };
  if (a.kv.code == KV8_E4M3) return off % 16 == 0 ? go(kv8_read_kernel<KV8_E4M3, 16>) : off % 8 == 0 ? go(kv8_read_kernel<KV8_E4M3, 8>) : go(kv8_read_kernel<KV8_E4M3, 1>);
  return off % 16 == 0 ? go(kv8_read_kernel<KV8_INT8, 16>) : off % 8 == 0 ? go(kv8_read_kernel<KV8_INT8, 8>) : go(kv8_read_kernel<KV8_INT8, 1>);
}

}  // namespace qie
