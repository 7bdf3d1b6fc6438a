// kv8_store.cu -- rotary positions of q and k and the store of k and v into a cache of 8 bits, one launch (qie_rope_store8), and its rows read back (qie_kv8_read).
//
// Positions as in rope_store.cu: turns in 64-bit fixed point, the hardware's sine and cosine.  Keys are turned in fp32 and coded from there, without a rounding to bf16 between.
// A warp takes a token and some of its heads, eight elements a lane, so that a head is 8 or 16 lanes: the lane's cosines and sines are computed once for all of them, a pair's other half is
// a shuffle away, and so is the largest element.  Bound by memory: every element is read and written once.
#include <algorithm>

#include "common.cuh"
#include "kernels.h"
#include "kv8.cuh"
#include "launch.h"

namespace qie {
namespace {

constexpr int THR = 256, WARPS = THR / 32;
enum { TURN_NONE, TURN_NEIGHBOURS, TURN_LANES, TURN_ANY };  // pairs: none; within a lane; of lanes half / 8 apart; of any elements

template <int HD, int CODE, int TURN, bool WIDE>
__global__ void __launch_bounds__(THR) rope_store8_kernel(Rope8Args a, int chunks, int per) {
  constexpr int LH = HD / 8, HW = 32 / LH;  // lanes of a head, heads of a warp at a time
  constexpr int NP = TURN == TURN_NEIGHBOURS ? 4 : TURN == TURN_NONE ? 1 : 8;  // pairs that the lane has a part of
  __shared__ bf16 s_row[TURN == TURN_ANY ? WARPS * HW * HD : 1];
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane / LH, p = lane % LH, e0 = p * 8;
  const int half = a.rotated / 2, n_kv = a.kv.n_kv, heads = a.n_q + 2 * n_kv;
  const long long all = (long long)a.n_tok * chunks;
  unsigned long long turns[NP];  // of the lane's pairs a position, their fraction in 2^-64
  bool on[NP];
  if constexpr (TURN != TURN_NONE) {
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      const int e = TURN == TURN_NEIGHBOURS ? e0 + 2 * j : e0 + j;
      on[j] = e < a.rotated;
      const double w = on[j] ? a.freq[TURN == TURN_NEIGHBOURS ? e / 2 : e < half ? e : e - half] * 0.15915494309189533577 : 0.0;
      turns[j] = (unsigned long long)((w - floor(w)) * 18446744073709551616.0);
    }
  }
  for (long long w = (long long)blockIdx.x * WARPS + warp; w < all; w += (long long)gridDim.x * WARPS) {
    const int t = (int)(w / chunks), chunk = (int)(w - (long long)t * chunks);
    const int pos = TURN == TURN_NONE ? 0 : a.pos[t], row = a.row[t];
    const bool kept = row >= 0 && row < a.kv.n_pages * a.kv.page_size;
    float c[NP], s[NP];
    if constexpr (TURN != TURN_NONE) {
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        const int at = (int)((unsigned long long)(unsigned)pos * turns[j] >> 32);  // from -1/2 of a turn on, in 2^-32
        __sincosf((float)at * 1.4629180792671596e-9f, &s[j], &c[j]);              // (2 pi / 2^32)
        c[j] = on[j] ? c[j] * a.factor : 1.f, s[j] = on[j] ? s[j] * a.factor : 0.f;
        if (TURN != TURN_NEIGHBOURS && e0 + j < half) s[j] = -s[j];
      }
    }
    for (int h0 = chunk * per; h0 < min(heads, chunk * per + per); h0 += HW) {
      const int head = h0 + sub;
      const int kind = head >= heads || head >= chunk * per + per ? -1 : head < a.n_q ? 0 : head < a.n_q + n_kv ? 1 : 2;
      if (__ballot_sync(0xffffffffu, kind == 0 ? pos >= 0 : kind > 0 && kept) == 0) continue;
      const int hk = head - a.n_q - (kind == 2 ? n_kv : 0);
      uint32_t x[4] = {0, 0, 0, 0};
      if (kind >= 0) {
        const bf16* src = kind == 0 ? a.q + (size_t)t * a.q_stride + (size_t)head * HD : kind == 1 ? a.k + (size_t)t * a.k_stride + (size_t)hk * HD : a.v + (size_t)t * a.v_stride + (size_t)hk * HD;
        src += e0;
        if constexpr (WIDE) {
          const uint4 v = *reinterpret_cast<const uint4*>(src);
          x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) x[j] = pack2(src[2 * j], src[2 * j + 1]);
        }
      }
      float y[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) y[2 * j] = lo2f(x[j]), y[2 * j + 1] = hi2f(x[j]);
      if constexpr (TURN == TURN_NEIGHBOURS) {
        if (kind < 2) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float u = y[2 * j], v = y[2 * j + 1];
            y[2 * j] = u * c[j] - v * s[j], y[2 * j + 1] = v * c[j] + u * s[j];
          }
        }
      } else if constexpr (TURN == TURN_LANES) {
        const int d = half / 8, from = e0 < half ? lane + d : e0 < a.rotated ? lane - d : lane;
        uint32_t o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = __shfl_sync(0xffffffffu, x[j], from);
        if (kind < 2) {
#pragma unroll
          for (int j = 0; j < 4; ++j) y[2 * j] = y[2 * j] * c[2 * j] + lo2f(o[j]) * s[2 * j], y[2 * j + 1] = y[2 * j + 1] * c[2 * j + 1] + hi2f(o[j]) * s[2 * j + 1];
        }
      } else if constexpr (TURN == TURN_ANY) {
        bf16* mine = s_row + (warp * HW + sub) * HD;
        __syncwarp();
        *reinterpret_cast<uint4*>(mine + e0) = make_uint4(x[0], x[1], x[2], x[3]);
        __syncwarp();
        if (kind < 2) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int e = e0 + j;
            if (e < a.rotated) y[j] = y[j] * c[j] + bf2f(mine[e < half ? e + half : e - half]) * s[j];
          }
        }
      }
      uint32_t most = 0;  // of the bits without signs: infinities and what is no number are above all numbers
#pragma unroll
      for (int j = 0; j < 8; ++j) most = max(most, __float_as_uint(y[j]) & 0x7fffffffu);
#pragma unroll
      for (int d = 1; d < LH; d <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, d));
      if (kind == 0) {
        if (pos < 0) continue;
        bf16* dst = a.q_out + (size_t)t * a.q_out_stride + (size_t)head * HD + e0;
        const uint4 v = make_uint4(pack2f(y[0], y[1]), pack2f(y[2], y[3]), pack2f(y[4], y[5]), pack2f(y[6], y[7]));
        if constexpr (WIDE) {
          *reinterpret_cast<uint4*>(dst) = v;
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) dst[j] = f2bf(y[j]);
        }
      } else if (kind > 0 && kept) {
        const uint32_t byte = kv8_scale_byte<CODE>(most);
        const float f = kv8_inverse(byte);
        const size_t vec = a.kv.vec(a.layer, kind - 1, hk, row);
        uint2 code = make_uint2(0, 0);
        if (byte != 255) code = make_uint2(kv8_pack<CODE>(y[0] * f, y[1] * f, y[2] * f, y[3] * f), kv8_pack<CODE>(y[4] * f, y[5] * f, y[6] * f, y[7] * f));
        *reinterpret_cast<uint2*>(a.kv.codes + vec * HD + e0) = code;
        if (p == 0) a.kv.scale[vec] = (uint8_t)byte;
      }
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
  const int heads = a.n_q + 2 * a.kv.n_kv, groups = (heads + HW - 1) / HW;
  const int want = std::min(groups, std::max(1, 16 * sms / a.n_tok)), per = (groups + want - 1) / want * HW, chunks = (heads + per - 1) / per;
  const long long warps = (long long)a.n_tok * chunks;
  const int ctas = (int)std::min<long long>((warps + WARPS - 1) / WARPS, 8ll * sms);
  if (wide) return launched(launch_k(rope_store8_kernel<HD, CODE, TURN, true>, dim3(ctas), dim3(THR), 0, st, a, chunks, per));
  return launched(launch_k(rope_store8_kernel<HD, CODE, TURN, false>, dim3(ctas), dim3(THR), 0, st, a, chunks, per));
}
template <int HD, int CODE>
cudaError_t launch_code(const Rope8Args& a, bool wide, cudaStream_t st) {
  if (!a.freq) return launch_turn<HD, CODE, TURN_NONE>(a, wide, st);
  if (a.neighbours) return launch_turn<HD, CODE, TURN_NEIGHBOURS>(a, wide, st);
  return a.rotated % 16 == 0 ? launch_turn<HD, CODE, TURN_LANES>(a, wide, st) : launch_turn<HD, CODE, TURN_ANY>(a, wide, st);
}

// sixteen elements a thread
template <int CODE, bool WIDE>
__global__ void __launch_bounds__(THR) kv8_read_kernel(Kv8ReadArgs a) {
  pdl_wait();
  pdl_trigger();
  const int hd = a.kv.hd, pieces = hd / 16, heads = a.kv.n_kv, per = 2 * heads * pieces;
  const long long all = (long long)a.n_rows * per;
  for (long long i = (long long)blockIdx.x * THR + threadIdx.x; i < all; i += (long long)gridDim.x * THR) {
    const int r = (int)(i / per), u = (int)(i - (long long)r * per), kv = u / (heads * pieces), head = (u - kv * heads * pieces) / pieces, piece = u % pieces;
    const int row = a.row[r];
    bf16* dst = kv ? a.v : a.k;
    if (!dst || row < 0 || row >= a.kv.n_pages * a.kv.page_size) continue;
    dst += (size_t)r * (kv ? a.v_stride : a.k_stride) + (size_t)head * hd + piece * 16;
    const size_t vec = a.kv.vec(a.layer, kv, head, row);
    const float f = kv8_scale(a.kv.scale[vec]);
    const uint4 code = *reinterpret_cast<const uint4*>(a.kv.codes + vec * hd + piece * 16);
    const uint32_t w[4] = {code.x, code.y, code.z, code.w};
    uint32_t o[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t lo, hi;
      kv8_unpack<CODE>(w[j], lo, hi);
      o[2 * j] = pack2f(h_lo(lo) * f, h_hi(lo) * f), o[2 * j + 1] = pack2f(h_lo(hi) * f, h_hi(hi) * f);
    }
    if constexpr (WIDE) {
      *reinterpret_cast<uint4*>(dst) = make_uint4(o[0], o[1], o[2], o[3]);
      *reinterpret_cast<uint4*>(dst + 8) = make_uint4(o[4], o[5], o[6], o[7]);
    } else {
      uint16_t* to = reinterpret_cast<uint16_t*>(dst);
#pragma unroll
      for (int j = 0; j < 8; ++j) to[2 * j] = (uint16_t)o[j], to[2 * j + 1] = (uint16_t)(o[j] >> 16);
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
  const long long items = (long long)a.n_rows * 2 * a.kv.n_kv * (a.kv.hd / 16);
  const dim3 grid((unsigned)std::min<long long>((items + THR - 1) / THR, 8ll * sms)), block(THR);
  const bool wide = off % 8 == 0;
  if (a.kv.code == KV8_E4M3) return launched(wide ? launch_k(kv8_read_kernel<KV8_E4M3, true>, grid, block, 0, st, a) : launch_k(kv8_read_kernel<KV8_E4M3, false>, grid, block, 0, st, a));
  return launched(wide ? launch_k(kv8_read_kernel<KV8_INT8, true>, grid, block, 0, st, a) : launch_k(kv8_read_kernel<KV8_INT8, false>, grid, block, 0, st, a));
}

}  // namespace qie
