// logit_rules.cu -- penalties for tokens that were there, biases and masks over rows of logits (qie_logits_process).
//
// A CTA takes a stretch of one row's vocabulary: it counts the row's tokens that lie in it (shared memory, whole numbers, so their order does not
// matter), adds up the biases of a token in the order of the list, and then passes once over the logits.
#include "common.cuh"
#include "kernels.h"
#include "launch.h"

namespace qie {
namespace {

constexpr int NTHR = 256, STRETCH = 4096;

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

template <typename T>
__global__ void __launch_bounds__(NTHR) logit_rules_kernel(LogitArgs a) {
  __shared__ uint32_t seen[STRETCH];   // generated ones; the top bit: in the list
  __shared__ uint32_t entry[STRETCH];  // the first bias of the token; the top bit: there are more
  __shared__ float bias[STRETCH];
  pdl_wait();
  pdl_trigger();
  const int row = blockIdx.y, lo = blockIdx.x * STRETCH, n = min(STRETCH, a.vocab - lo), tid = threadIdx.x;
  for (int i = tid; i < n; i += NTHR) seen[i] = 0, entry[i] = 0x7fffffffu, bias[i] = 0.f;
  __syncthreads();
  if (a.tok_start) {
    const int2 s = span(a.tok_start, row, a.n_tokens);
    const int gen = a.gen_start ? a.gen_start[row] : s.x;
    for (int j = s.x + tid; j < s.y; j += NTHR) {
      const unsigned i = (unsigned)a.tokens[j] - (unsigned)lo;
      if (i < (unsigned)n) {
        if (j >= gen) atomicAdd(&seen[i], 1u);
        else atomicOr(&seen[i], 0x80000000u);
      }
    }
  }
  if (a.bias_start) {
    const int2 s = span(a.bias_start, row, a.n_bias);
    for (int j = s.x + tid; j < s.y; j += NTHR) {
      const unsigned i = (unsigned)a.bias_ids[j] - (unsigned)lo;
      if (i < (unsigned)n) atomicMin(&entry[i], (uint32_t)j);
    }
    __syncthreads();
    for (int j = s.x + tid; j < s.y; j += NTHR) {
      const unsigned i = (unsigned)a.bias_ids[j] - (unsigned)lo;
      if (i < (unsigned)n && (entry[i] & 0x7fffffffu) != (uint32_t)j) atomicOr(&entry[i], 0x80000000u);
    }
    __syncthreads();
    for (int j = s.x + tid; j < s.y; j += NTHR) {
      const int id = a.bias_ids[j];
      const unsigned i = (unsigned)id - (unsigned)lo;
      if (i < (unsigned)n && (entry[i] & 0x7fffffffu) == (uint32_t)j) {
        float sum = a.bias[j];
        if (entry[i] >> 31)
          for (int k = j + 1; k < s.y; ++k)
            if (a.bias_ids[k] == id) sum += a.bias[k];
        bias[i] = sum;
      }
    }
  }
  __syncthreads();
  const float rep = a.repetition ? a.repetition[row] : 1.f, pres = a.presence ? a.presence[row] : 0.f, freq = a.frequency ? a.frequency[row] : 0.f;
  const int m = a.mask ? (a.mask_row ? a.mask_row[row] : row) : -1;
  const uint32_t* mask = m >= 0 && m < a.n_masks ? a.mask + (size_t)m * a.mask_words : nullptr;
  const T* in = (const T*)a.in + (size_t)row * a.stride + lo;
  T* out = (T*)a.out + (size_t)row * a.out_stride + lo;
  for (int i = tid; i < n; i += NTHR) {
    float x = load(in + i);
    const uint32_t w = seen[i], times = w & 0x7fffffffu;
    if (w && a.repetition) x = x > 0.f ? x / rep : x * rep;
    if (times) {
      x -= freq * (float)times;
      x -= pres;
    }
    x += bias[i];
    if (mask && !(mask[(lo + i) >> 5] >> ((lo + i) & 31) & 1)) x = -INFINITY;
    store(out + i, x);
  }
}

}  // namespace

cudaError_t launch_logit_rules(const LogitArgs& a, cudaStream_t st) {
  const dim3 grid((a.vocab + STRETCH - 1) / STRETCH, a.n_rows);
  return launched(a.f32 ? launch_k(logit_rules_kernel<float>, grid, dim3(NTHR), 0, st, a) : launch_k(logit_rules_kernel<bf16>, grid, dim3(NTHR), 0, st, a));
}

}  // namespace qie
