// logit_rules.cu -- penalties for tokens that were there, biases and masks over rows of logits (qie_logits_process).
//
// A CTA takes a stretch of one row's vocabulary.  It passes the logits through, 16 bytes at a time, with the mask; beside that it reads the row's lists and
// counts, in shared memory, how often they have each token of the stretch (whole numbers, so the order does not matter).  The first one to meet a token notes
// it, and at the end the noted tokens, few of the stretch, are computed from the input and written over what was passed through.  A token with several
// biases gets their sum in the order of the list.
#include "common.cuh"
#include "kernels.h"
#include "launch.h"

namespace qie {
namespace {

// a token's word: how often it is among the generated ones, and
constexpr uint32_t LISTED = 1u << 31, BIASED = 1u << 30, MORE = 1u << 29, TIMES = MORE - 1;  // in the row's list; has a bias; has several
constexpr uint32_t NONE = 0x7fffffffu;

template <typename T>
__device__ __forceinline__ float load(const T* p) {
  if constexpr (sizeof(T) == 2) return bf2f(*p);
  else return *p;
}
template <typename T>
__device__ __forceinline__ void store(T* p, float v) {
  if constexpr (sizeof(T) == 2) *p = f2bf(v);
  else *p = v;
}
// [from, to) of a list of n, whatever the offsets say
__device__ __forceinline__ int2 span(const int* start, int i, int n) {
  const int from = min(max(start[i], 0), n);
  return make_int2(from, min(max(start[i + 1], from), n));
}
// f(index, value) for a thread's share of p[s.x .. s.y), 16 bytes at a time
template <typename F>
__device__ __forceinline__ void each(const int* p, int2 s, F f) {
  int from = s.x;
  const int lead = (int)((16 - (reinterpret_cast<uintptr_t>(p + s.x) & 15)) & 15) / 4, head = min(s.y, s.x + lead);
  if ((int)threadIdx.x < head - from) f(from + threadIdx.x, p[from + threadIdx.x]);
  from = head;
  const int quads = (s.y - from) / 4;
  for (int q = threadIdx.x; q < quads; q += blockDim.x) {
    const int4 v = *reinterpret_cast<const int4*>(p + from + 4 * q);
    f(from + 4 * q, v.x), f(from + 4 * q + 1, v.y), f(from + 4 * q + 2, v.z), f(from + 4 * q + 3, v.w);
  }
  from += 4 * quads;
  if ((int)threadIdx.x < s.y - from) f(from + threadIdx.x, p[from + threadIdx.x]);
}

// G groups of 16 bytes a thread.  A stretch begins on a 16-byte boundary of the row's input, so `shift` elements ahead of where a row on a boundary had it.
template <typename T, int THR, int G>
__global__ void __launch_bounds__(THR) logit_rules_kernel(LogitArgs a) {
  constexpr int E = 16 / sizeof(T), STRETCH = G * THR * E;
  extern __shared__ __align__(16) uint32_t seen[];  // [STRETCH], then (16 bits each) the noted tokens, then, where there are biases, the first one of each token
  uint16_t* noted = reinterpret_cast<uint16_t*>(seen + STRETCH);
  uint32_t* entry = seen + STRETCH + STRETCH / 2;
  __shared__ int n_noted;
  pdl_wait();
  pdl_trigger();
  const int row = blockIdx.y, tid = threadIdx.x;
  const T* in = (const T*)a.in + (size_t)row * a.stride;
  T* out = (T*)a.out + (size_t)row * a.out_stride;
  const int shift = (int)((reinterpret_cast<uintptr_t>(in) & 15) / sizeof(T)), lo = blockIdx.x * STRETCH - shift;
  const bool out16 = ((reinterpret_cast<uintptr_t>(out) / sizeof(T) - shift) * sizeof(T) & 15) == 0;
  const int m = a.mask ? (a.mask_row ? a.mask_row[row] : row) : -1;
  const uint32_t* mask = m >= 0 && m < a.n_masks ? a.mask + (size_t)m * a.mask_words : nullptr;
  auto allowed = [&](int t) { return !mask || (mask[t >> 5] >> (t & 31) & 1); };
  uint4 x[G];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const int t = lo + (g * THR + tid) * E;
    if (t >= 0 && t + E <= a.vocab) x[g] = *reinterpret_cast<const uint4*>(in + t);
  }
  const bool biases = a.bias_start != nullptr, lists = a.tok_start != nullptr;
  if (lists || biases)
    for (int i = tid; i < STRETCH / 4; i += THR) {
      reinterpret_cast<uint4*>(seen)[i] = make_uint4(0, 0, 0, 0);
      if (biases) reinterpret_cast<uint4*>(entry)[i] = make_uint4(NONE, NONE, NONE, NONE);
    }
  if (tid == 0) n_noted = 0;
  __syncthreads();
  auto note = [&](unsigned i, uint32_t before) {
    if (before == 0) noted[atomicAdd(&n_noted, 1)] = (uint16_t)i;
  };
  if (lists) {
    const int2 s = span(a.tok_start, row, a.n_tokens);
    const int gen = a.gen_start ? a.gen_start[row] : s.x;
    each(a.tokens, s, [&](int j, int id) {
      const unsigned i = (unsigned)id - (unsigned)lo;
      if (i < (unsigned)STRETCH && (unsigned)id < (unsigned)a.vocab) note(i, j >= gen ? atomicAdd(&seen[i], 1u) : atomicOr(&seen[i], LISTED));
    });
  }
  const int2 bs = biases ? span(a.bias_start, row, a.n_bias) : make_int2(0, 0);
  if (biases)
    each(a.bias_ids, bs, [&](int j, int id) {
      const unsigned i = (unsigned)id - (unsigned)lo;
      if (i < (unsigned)STRETCH && (unsigned)id < (unsigned)a.vocab) {
        const bool more = atomicMin(&entry[i], (uint32_t)j) != NONE;
        note(i, atomicOr(&seen[i], more ? BIASED | MORE : BIASED));
      }
    });
  // ---- the logits with the mask
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const int t0 = lo + (g * THR + tid) * E;
    if (t0 >= a.vocab || t0 + E <= 0) continue;
    if (t0 >= 0 && t0 + E <= a.vocab) {
      uint32_t* w = reinterpret_cast<uint32_t*>(&x[g]);
      if (mask) {
        const uint32_t bits = __funnelshift_r(mask[t0 >> 5], mask[(t0 + E - 1) >> 5], t0 & 31);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const bool no = !(bits >> e & 1);
          if constexpr (sizeof(T) == 4) w[e] = no ? 0xff800000u : w[e];
          else w[e / 2] = no ? (e & 1 ? (w[e / 2] & 0xffffu) | 0xff800000u : (w[e / 2] & 0xffff0000u) | 0xff80u) : w[e / 2];
        }
      }
      if (out16) {
        *reinterpret_cast<uint4*>(out + t0) = x[g];
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          if constexpr (sizeof(T) == 4) out[t0 + e] = __uint_as_float(w[e]);
          else out[t0 + e] = __ushort_as_bfloat16((unsigned short)(w[e / 2] >> (e & 1 ? 16 : 0)));
        }
      }
    } else {
      for (int t = max(t0, 0); t < min(t0 + E, a.vocab); ++t) out[t] = allowed(t) ? in[t] : (T)(-INFINITY);
    }
  }
  if (!lists && !biases) return;
  __syncthreads();
  // ---- the noted tokens.  (In place: their logits are as they were, or masked.)
  const float rep = a.repetition ? a.repetition[row] : 1.f, pres = a.presence ? a.presence[row] : 0.f, freq = a.frequency ? a.frequency[row] : 0.f;
  for (int k = tid; k < n_noted; k += THR) {
    const int i = noted[k], id = lo + i;
    if (!allowed(id)) continue;
    const uint32_t w = seen[i], times = w & TIMES;
    float v = load(in + id);
    if ((times || w & LISTED) && a.repetition) v = v > 0.f ? v / rep : v * rep;
    if (times) {
      v -= freq * (float)times;
      v -= pres;
    }
    if (w & BIASED) {
      const int j = (int)entry[i];
      float sum = a.bias[j];
      if (w & MORE)
        for (int n = j + 1; n < bs.y; ++n)
          if (a.bias_ids[n] == id) sum += a.bias[n];
      v += sum;
    }
    store(out + id, v);
  }
}

template <typename T, int THR, int G>
cudaError_t launch_g(const LogitArgs& a, cudaStream_t st) {
  constexpr int E = 16 / sizeof(T), STRETCH = G * THR * E;
  static_assert(STRETCH <= 65536, "noted in 16 bits");
  static PerDeviceOnce set;
  if (set.need()) {
    const cudaError_t e = cudaFuncSetAttribute(logit_rules_kernel<T, THR, G>, cudaFuncAttributeMaxDynamicSharedMemorySize, STRETCH * 10);
    if (e != cudaSuccess) return e;
    set.done();
  }
  const dim3 grid((a.vocab + E - 2) / STRETCH + 1, a.n_rows);
  return launched(launch_k(logit_rules_kernel<T, THR, G>, grid, dim3(THR), a.bias_start ? STRETCH * 10 : a.tok_start ? STRETCH * 6 : 0, st, a));
}

}  // namespace

cudaError_t launch_logit_rules(const LogitArgs& a, cudaStream_t st) {
  // one row: as many CTAs as share it out over the chip; many: stretches that read a row's lists less often
  const bool few = (long long)a.n_rows * a.vocab < 148ll * 4096;
  if (a.f32) return few ? launch_g<float, 256, 1>(a, st) : launch_g<float, 512, 4>(a, st);
  return few ? launch_g<bf16, 128, 1>(a, st) : launch_g<bf16, 512, 2>(a, st);
}

}  // namespace qie
