// logit_rules.cu -- penalties for tokens that were there, biases and masks over rows of logits (qie_logits_process).
//
// A CTA has a share of one row's vocabulary, chunks of 256 tokens in turn with the row's other CTAs (frequent tokens have low numbers).  It starts copies of all its
// chunks into shared memory; while they are on their way it reads the row's lists and collects the share's tokens in a hash table: how often a token is there (whole
// numbers, so their order does not matter) and the first entry of its biases.  Then those tokens, a few thousand of a row, are computed in the chunks, and the chunks are
// written out, masked.  A token with several biases gets their sum in the order of the list.  In place, a row without a mask has its tokens computed where they are.
// Bound by memory as far as the lists go: 64 rows of 151936 bf16 are 39 MB; B200, in a graph with inputs that are not in L2, the copy alone 9.2 us, with masks 10.6, with lists of
// 4000 tokens 14.5, with 300 biases a row and masks for half of them 17.8, of which the tokens of the lists are a chain of latencies (their numbers, the table, the logits).  One
// row of fp32 3.6.
#include <algorithm>

#include "common.cuh"
#include "kernels.h"
#include "launch.h"

namespace qie {
namespace {

constexpr int THR = 512, CHUNK_BITS = 8;
constexpr int SLOT_BITS = 11, SLOTS = 1 << SLOT_BITS, MOST_PROBES = 64, MOST_SHARE = 6, TILE_BYTES = 80 * 1024;
constexpr int FEW = 4;  // of a warp's tokens
constexpr uint32_t EMPTY = 0xffffffffu, NONE = 0x7fffffffu, PLACE = 1u << 31;
// a token's word: how often it is among the generated ones, and
constexpr uint32_t LISTED = 1u << 31, BIASED = 1u << 30, MORE = 1u << 29, TIMES = MORE - 1;  // in the row's list; has a bias; has several

// [from, to) of a list of n, whatever the offsets say
__device__ __forceinline__ int2 span(const int* start, int i, int n) {
  const int from = min(max(start[i], 0), n);
  return make_int2(from, min(max(start[i + 1], from), n));
}
// a thread's next tokens of a list, U of them in steps of the CTA's threads; those behind the end are -1
template <int U>
struct Next {
  int id[U];
  __device__ __forceinline__ Next(const int* p, int2 s, int at) {
#pragma unroll
    for (int u = 0; u < U; ++u) id[u] = at + u * THR < s.y - s.x ? p[s.x + at + u * THR] : -1;
  }
  // hit(place in the list, token) for those that are `mine`: a warp goes round as often as one of its threads has some
  template <typename M, typename F>
  __device__ __forceinline__ void each(int at, M mine, F hit) const {
    unsigned hits = 0;
#pragma unroll
    for (int u = 0; u < U; ++u) hits |= (unsigned)mine(id[u]) << u;
    for (; hits; hits &= hits - 1) {
      const int u = __ffs(hits) - 1;
      int x = id[0];
#pragma unroll
      for (int e = 1; e < U; ++e) x = u == e ? id[e] : x;
      hit(at + u * THR, x);
    }
  }
};
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
constexpr int CHUNK = 1 << CHUNK_BITS, CHUNK_WORDS = CHUNK / 32 + 1;  // mask words that a chunk at any place touches
template <typename T>
constexpr size_t chunk_bytes = CHUNK * sizeof(T) + CHUNK_WORDS * 4;

// CTA y of 2^share of a row has the chunks whose number's lowest `share` bits are y.  Chunks begin on 16-byte boundaries of the row's input, so `shift` elements ahead
// of where a row on a boundary has them.
template <typename T>
__global__ void __launch_bounds__(THR) logit_rules_kernel(LogitArgs a, int share, int most) {  // most: chunks that a CTA has at most
  constexpr int E = 16 / sizeof(T), GROUPS = CHUNK / E;  // 16-byte groups of a chunk
  extern __shared__ __align__(16) unsigned char tile[];
  __shared__ __align__(16) uint32_t key[SLOTS], word[SLOTS], entry[SLOTS];  // the token, its word, the first of its biases
  __shared__ uint16_t used[SLOTS];  // the slots in use
  __shared__ int full, n_used;
  pdl_wait();
  pdl_trigger();
  const int row = blockIdx.x, tid = threadIdx.x;
  const T* in = (const T*)a.in + (size_t)row * a.stride;
  T* out = (T*)a.out + (size_t)row * a.out_stride;
  const int shift = (int)((reinterpret_cast<uintptr_t>(in) & 15) / sizeof(T));
  const bool lists = a.tok_start || a.bias_start;
  int depth = share;
  unsigned low = blockIdx.y;
  // Tokens of the class (depth, low): the lowest `depth` bits of the place, its chunk's number first.  A class that finds no room in the table is taken in halves; at the
  // latest one with no more tokens than probes fits.
  auto place = [&](int id) { return __funnelshift_r((unsigned)(id + shift), (unsigned)(id + shift), CHUNK_BITS); };
  auto mine = [&](int id) { return (unsigned)id < (unsigned)a.vocab && (place(id) & ((1u << depth) - 1)) == low; };
  auto slot_at = [&](int id) { return (place(id) >> depth) * 2654435769u >> (32 - SLOT_BITS); };
  auto slot_of = [&](int id) {  // below 0: there is none
    unsigned k = slot_at(id);
    for (int n = 0; n < MOST_PROBES; ++n, k = (k + 1) & (SLOTS - 1)) {
      const uint32_t have = atomicCAS(&key[k], EMPTY, (uint32_t)id);
      if (have == EMPTY || have == (uint32_t)id) return (int)k;
    }
    full = 1;
    return -1;
  };
  auto clear = [&] {
    for (int i = tid; i < SLOTS / 4; i += THR) {
      reinterpret_cast<uint4*>(key)[i] = make_uint4(EMPTY, EMPTY, EMPTY, EMPTY);
      reinterpret_cast<uint4*>(word)[i] = make_uint4(0, 0, 0, 0);
      reinterpret_cast<uint4*>(entry)[i] = make_uint4(NONE, NONE, NONE, NONE);
    }
    if (tid == 0) full = n_used = 0;
  };
  // ---- the chunks into shared memory, and the words of the mask
  const bool copy = a.in != a.out;
  const int chunks = (((a.vocab + shift + CHUNK - 1) >> CHUNK_BITS) - (int)blockIdx.y + (1 << share) - 1) >> share;
  uint32_t* words = reinterpret_cast<uint32_t*>(tile + (size_t)most * CHUNK * sizeof(T));  // [chunk][CHUNK_WORDS]
  auto first_of = [&](int c) { return (((c << share) + (int)blockIdx.y) << CHUNK_BITS) - shift; };  // the chunk's first token
  auto read = [&] {
    for (int g = tid; g < chunks * GROUPS; g += THR) {
      const int c = g / GROUPS, t0 = first_of(c) + (g - c * GROUPS) * E;
      T* to = reinterpret_cast<T*>(tile) + (size_t)g * E;
      if (t0 >= 0 && t0 + E <= a.vocab) cp_async16(smem_u32(to), in + t0);
      else
        for (int e = 0; e < E; ++e)
          if (t0 + e >= 0 && t0 + e < a.vocab) to[e] = in[t0 + e];
    }
    cp_async_commit();
  };
  // (numbers that lists and masks hang on, ahead of the copies)
  const int2 ts = a.tok_start ? span(a.tok_start, row, a.n_tokens) : make_int2(0, 0), bs = a.bias_start ? span(a.bias_start, row, a.n_bias) : make_int2(0, 0);
  const int gen = (a.gen_start && a.tok_start ? a.gen_start[row] : ts.x) - ts.x;
  const float rep = a.repetition ? a.repetition[row] : 1.f, pres = a.presence ? a.presence[row] : 0.f, freq = a.frequency ? a.frequency[row] : 0.f;
  const int m = a.mask ? (a.mask_row ? a.mask_row[row] : row) : -1;
  if (copy) read();
  const uint32_t* mask = m >= 0 && m < a.n_masks ? a.mask + (size_t)m * a.mask_words : nullptr;
  const bool staged = copy || mask;
  if (!copy && mask) read();
  // ---- the lists
  constexpr int UT = 8, UB = 1;
  auto collect = [&](auto&& ready) {  // `ready` between the loads and their use
    Next<UT> t(a.tokens, ts, tid);
    Next<UB> b(a.bias_ids, bs, tid);
    if (tid < bs.y - bs.x) asm volatile("prefetch.global.L2 [%0];" ::"l"(a.bias + bs.x + tid));
    ready();
    for (int i = tid;;) {
      t.each(i, mine, [&](int j, int id) {
        const int k = slot_of(id);
        if (k < 0) return;
        if (j >= gen) atomicAdd(&word[k], 1u);
        else atomicOr(&word[k], LISTED);
      });
      if (ts.y - ts.x - i <= UT * THR) break;
      i += UT * THR;
      t = Next<UT>(a.tokens, ts, i);
    }
    for (int i = tid;;) {
      b.each(i, mine, [&](int j, int id) {
        const int k = slot_of(id);
        if (k >= 0) atomicOr(&word[k], atomicMin(&entry[k], (uint32_t)j) != NONE ? BIASED | MORE : BIASED);
      });
      if (bs.y - bs.x - i <= UB * THR) break;
      i += UB * THR;
      b = Next<UB>(a.bias_ids, bs, i);
    }
  };
  if (lists)
    collect([&] {
      clear();
      __syncthreads();
    });
  if (mask)
    for (int i = tid; i < chunks * CHUNK_WORDS; i += THR) {
      const int c = i / CHUNK_WORDS, w = (first_of(c) >> 5) + i - c * CHUNK_WORDS;
      words[i] = w >= 0 && w < (a.vocab + 31) >> 5 ? mask[w] : 0;
    }
  if (staged) cp_async_wait<0>();
  __syncthreads();
  // ---- the tokens of the lists
  auto place_of = [&](int id) {  // in the chunks
    const int v = id + shift;
    return ((v >> (CHUNK_BITS + share)) << CHUNK_BITS) + (v & (CHUNK - 1));
  };
  while (lists) {
    if (full) {
      ++depth;
    } else {
      // the slots in use, side by side
      constexpr int MINE = SLOTS / THR;
      unsigned have[MINE];
      int before = 0;
#pragma unroll
      for (int i = 0; i < MINE; ++i) have[i] = __ballot_sync(0xffffffffu, key[i * THR + tid] != EMPTY), before += __popc(have[i]);
      if ((tid & 31) == 0) before = atomicAdd(&n_used, before);
      before = __shfl_sync(0xffffffffu, before, 0);
#pragma unroll
      for (int i = 0; i < MINE; ++i) {
        if (have[i] >> (tid & 31) & 1) used[before + __popc(have[i] & ((1u << (tid & 31)) - 1))] = (uint16_t)(i * THR + tid);
        before += __popc(have[i]);
      }
      __syncthreads();
      const int lane = tid & 31;
      for (int first = tid - lane; first < n_used; first += THR) {
        const bool some = first + lane < n_used;
        const int k = used[some ? first + lane : first], id = (int)key[k], j = (int)entry[k];
        const uint32_t w = word[k], times = w & TIMES;
        T* at = staged ? reinterpret_cast<T*>(tile) + place_of(id) : out + id;
        float v = load(at), sum = w & BIASED ? a.bias[bs.x + j] : 0.f;
        // Several biases of a token: the warp reads the list once for all of its tokens that have some, from the first one's first on, and adds those of each in their order.  A few
        // tokens are compared one after the other with 32 biases; where there are more, their slots get their places among those in use, and a bias finds its token by the table.
        // (64 rows.  300 biases, a handful of tokens with several: 17.8 us, all by the table 21.1; 5000 tokens, each twice: 520, all one after the other 2130, and 5300 with the list
        // read for each.)
        if (const unsigned more = __ballot_sync(0xffffffffu, some && w & MORE)) {
          const bool own = more >> lane & 1, many = __popc(more) > FEW;
          if (own) sum = 0.f;
          if (many && own) entry[k] = PLACE + first + lane;
          __syncwarp();
          for (int i = bs.x + __reduce_min_sync(0xffffffffu, own ? j : 0x7fffffff); i < bs.y; i += 32) {
            const int x = i + lane < bs.y ? a.bias_ids[i + lane] : -1;
            const float b = i + lane < bs.y ? a.bias[i + lane] : 0.f;
            if (many) {
              unsigned to = 32;
              if (mine(x)) {
                unsigned q = slot_at(x);
                for (int n = 1; n < MOST_PROBES && key[q] != (uint32_t)x; ++n) q = (q + 1) & (SLOTS - 1);  // (all tokens of the class are there)
                to = entry[q] - (PLACE + first);
              }
              for (unsigned its = __ballot_sync(0xffffffffu, to < 32); its; its &= its - 1) {
                const int from = __ffs(its) - 1;
                const unsigned t = __shfl_sync(0xffffffffu, to, from);
                const float v = __shfl_sync(0xffffffffu, b, from);
                if (lane == t) sum += v;
              }
            } else {
              for (unsigned m = more; m; m &= m - 1) {
                const int from = __ffs(m) - 1;
                for (unsigned its = __ballot_sync(0xffffffffu, x == __shfl_sync(0xffffffffu, id, from)); its; its &= its - 1) {
                  const float v = __shfl_sync(0xffffffffu, b, __ffs(its) - 1);
                  if (lane == from) sum += v;
                }
              }
            }
          }
        }
        if ((times || w & LISTED) && a.repetition) v = v > 0.f ? v / rep : v * rep;
        if (times) {
          v -= freq * (float)times;
          v -= pres;
        }
        if (w & BIASED) v += sum;
        if (some) store(at, v);
      }
      // the next class
      while (depth > share && (low >> (depth - 1) & 1)) --depth, low &= (1u << depth) - 1;
      if (depth == share) break;
      low |= 1u << (depth - 1);
    }
    __syncthreads();
    clear();
    __syncthreads();
    collect([] {});
    __syncthreads();
  }
  if (!staged) return;
  __syncthreads();
  // ---- the chunks out
  const bool out16 = ((reinterpret_cast<uintptr_t>(out) / sizeof(T) - shift) * sizeof(T) & 15) == 0;
  for (int g = tid; g < chunks * GROUPS; g += THR) {
    const int c = g / GROUPS, first = first_of(c), t0 = first + (g - c * GROUPS) * E;
    uint4 x = *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(tile) + (size_t)g * E);
    uint32_t* w = reinterpret_cast<uint32_t*>(&x);
    if (mask) {
      const uint32_t* p = words + c * CHUNK_WORDS + (t0 >> 5) - (first >> 5);
      const uint32_t bits = (t0 & 31) + E <= 32 ? *p >> (t0 & 31) : __funnelshift_r(p[0], p[1], t0 & 31);
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int e = 0; e < E; ++e) w[e] = bits >> e & 1 ? w[e] : 0xff800000u;
      } else {
#pragma unroll
        for (int e = 0; e < E / 2; ++e) {  // a pair's bits as 16 bits each
          const uint32_t two = bits >> (2 * e), keep = ((two & 1) | (two & 2) << 15) * 0xffffu;
          w[e] = (w[e] & keep) | (0xff80ff80u & ~keep);
        }
      }
    }
    if (out16 && t0 >= 0 && t0 + E <= a.vocab) {
      *reinterpret_cast<uint4*>(out + t0) = x;
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if (t0 + e < 0 || t0 + e >= a.vocab) continue;
        if constexpr (sizeof(T) == 4) out[t0 + e] = __uint_as_float(w[e]);
        else out[t0 + e] = __ushort_as_bfloat16((unsigned short)(w[e / 2] >> (e & 1 ? 16 : 0)));
      }
    }
  }
}

template <typename T>
cudaError_t launch_t(const LogitArgs& a, cudaStream_t st) {
  if (!a.mask && a.in == a.out && !a.tok_start && !a.bias_start) return cudaSuccess;
  static PerDeviceOnce set;
  if (set.need()) {
    const cudaError_t e = cudaFuncSetAttribute(logit_rules_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, TILE_BYTES);
    if (e != cudaSuccess) return e;
    set.done();
  }
  int share = 0, dev = 0;
  const cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const bool staged = a.mask || a.in != a.out;
  const long long chunks = ((long long)a.vocab + 16 / sizeof(T) + CHUNK - 1) >> CHUNK_BITS;
  auto most = [&] { return (chunks + (1 << share) - 1) >> share; };  // of a CTA
  // CTAs a row: as many as their chunks need for room, two CTAs an SM, then as many as find room at once (64 rows by 4 CTAs 18.0 us, by 8 18.9)
  while (staged && most() * chunk_bytes<T> > TILE_BYTES) ++share;
  while (share < MOST_SHARE && (a.n_rows << (share + 1)) <= 2 * device_attribute<cudaDevAttrMultiProcessorCount>(dev)) ++share;
  return launched(launch_k(logit_rules_kernel<T>, dim3(a.n_rows, 1 << share), dim3(THR), staged ? most() * chunk_bytes<T> : 0, st, a, share, (int)most()));
}

}  // namespace

cudaError_t launch_logit_rules(const LogitArgs& a, cudaStream_t st) { return a.f32 ? launch_t<float>(a, st) : launch_t<bf16>(a, st); }

}  // namespace qie
