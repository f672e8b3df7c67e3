// Penalties for repeated tokens, biases and a grammar's mask on the logits of a decode step, with the greedy pick.
// For token v of a row, x its logit, r / f / p the row's penalties:
//   v in the history:                 x = x > 0 ? x / r : x * r
//   c times in what was generated:    x = x - f * c,  and x = x - p when c > 0
//   biases b of v:                    x = x + sum b
//   the mask's bit is 0:              x = -inf
// in fp32 in this order, rounded once to the logits' type.
#include <atomic>

#include "mkb_common.cuh"

namespace mkb {
namespace {

struct LogitArguments {
  const void* logits;
  void* out;
  const void* tokens;            // int32 or int64 [M, ...]
  const int* lengths;
  const int* prompts;
  const float* repetition;
  const float* frequency;
  const float* presence;
  const int* bias_tokens;
  const float* bias;
  const int* mask;
  unsigned long long* best;
  long long* picked;
  int64_t logits_stride, out_stride, tokens_stride, bias_stride, mask_words, mask_stride, offset;
  int width, history, biases, long_tokens, slice, widest, slots;    // widest: tokens of the longest chunk
};

// What bounds it: for many rows the logits, read and written once (4 bytes a token in 16 bits); for few, the chain of
// launch, history and one reduction.  So a row is spread over a cluster of CTAs, as many as keep the GPU busy, each with a
// slice of the vocabulary.  A CTA reads the whole history, gathers the slice's tokens with their counts in a hash table
// in shared memory (no [rows, vocabulary] state exists anywhere) and marks them in a bit map, while its first logits are
// under way.  Then the slice passes in 16-byte pieces as it is, masked in its own type, but for the marked tokens, and the
// greedy pick looks at a piece's maximum only; the marked tokens follow from the table's list, one a thread.  The CTAs' best
// words meet in the first one's shared memory, since an order of (value, lower token) does not depend on who comes first.
// Measured for 128 rows of 128256 tokens with 4000 in the history, 300 biases and a mask: penalties worked out where a piece
// met them 115 us (almost every warp did all of it for all of its tokens), a count per token in shared memory, chunk by chunk,
// 77 us, counts of the history's shares added into the other CTAs' memory 96 us (common tokens queued there), this form 41 to 45:
// 15 for the copy, 5 for the mask, 14 for the history, 10 for the biases.  One row with 300 tokens of history takes 5.
constexpr int kLogitThreads = 512;
constexpr int kDeep = 2;                  // pieces of a thread under way
constexpr int kSlots = 8192;              // of the hash table, at most; a power of two
constexpr int kMost = 6144;               // tokens it takes, three quarters of its slots; a longer history goes by chunks of a block
constexpr int kRanks = 16;                // CTAs of a row, at most
constexpr uint32_t kBiased = 0x80000000u; // of a count: the token has a bias
constexpr uint32_t kSeen = 0x40000000u;   // of a count with kBiased: the token is in the history, as all without it are
constexpr uint32_t kCount = kSeen - 1;    // how often it was generated
constexpr uint32_t kNoPlace = 0xffffffffu;
constexpr int64_t kNothing = -(int64_t(1) << 40);
constexpr int kBiases = 512;              // entries of a chunk that are listed in shared memory

template <typename T> struct Logit;
template <> struct Logit<float> {
  static constexpr int kVector = 4;
  static __device__ __forceinline__ float widen(float v) { return v; }
  static __device__ __forceinline__ float narrow(float v) { return v; }
  // A monotone map of values to unsigned words: NaN below everything, a negative zero as zero.
  static __device__ __forceinline__ uint32_t key(float v) {
    const uint32_t bits = __float_as_uint(v);
    if ((bits & 0x7fffffffu) > 0x7f800000u) return 0u;
    if (bits == 0x80000000u) return 0x80000000u;
    return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
  }
  static __device__ __forceinline__ float largest(const uint4& v) {
    return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
  }
  static constexpr uint32_t kLow = 0xff800000u, kNone = 0x7fffffffu;      // -inf, a NaN
  static __device__ __forceinline__ void mask(uint4& v, uint32_t bits, uint32_t other) {
    v.x = bits & 1u ? v.x : other; v.y = bits & 2u ? v.y : other;
    v.z = bits & 4u ? v.z : other; v.w = bits & 8u ? v.w : other;
  }
};
// fp16 and bf16: the 16-bit keys of the arg-max kernel, so that their words compare.
__device__ __forceinline__ uint32_t key16(uint32_t bits, uint32_t infinity) {
  if ((bits & 0x7fffu) > infinity) return 0u;
  if (bits == 0x8000u) return 0x8000u;
  return bits & 0x8000u ? ~bits & 0xffffu : bits | 0x8000u;
}
// Eight 16-bit values, those whose bit is 0 replaced by `other`.
__device__ __forceinline__ void mask16(uint4& v, uint32_t bits, uint32_t other) {
  // four bits to four bytes of ones or zeros (the factor puts bit i at bit 8i), each byte doubled
  const uint32_t low = ((bits & 15u) * 0x204081u & 0x1010101u) * 255u, high = ((bits >> 4 & 15u) * 0x204081u & 0x1010101u) * 255u;
  const uint32_t keep[4] = {__byte_perm(low, 0u, 0x1100), __byte_perm(low, 0u, 0x3322), __byte_perm(high, 0u, 0x1100), __byte_perm(high, 0u, 0x3322)};
  v.x = (v.x & keep[0]) | (other & ~keep[0]);
  v.y = (v.y & keep[1]) | (other & ~keep[1]);
  v.z = (v.z & keep[2]) | (other & ~keep[2]);
  v.w = (v.w & keep[3]) | (other & ~keep[3]);
}
template <> struct Logit<__half> {
  static constexpr int kVector = 8;
  static __device__ __forceinline__ float widen(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half narrow(float v) { return __float2half_rn(v); }
  static __device__ __forceinline__ uint32_t key(__half v) { return key16(__half_as_ushort(v), 0x7c00u); }
  static __device__ __forceinline__ __half largest(const uint4& v) {
    const __half2* h = reinterpret_cast<const __half2*>(&v);
    const __half2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return __hmax(__low2half(m), __high2half(m));
  }
  static constexpr uint32_t kLow = 0xfc00fc00u, kNone = 0x7fff7fffu;
  static __device__ __forceinline__ void mask(uint4& v, uint32_t bits, uint32_t other) { mask16(v, bits, other); }
};
template <> struct Logit<__nv_bfloat16> {
  static constexpr int kVector = 8;
  static __device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 narrow(float v) { return __float2bfloat16_rn(v); }
  static __device__ __forceinline__ uint32_t key(__nv_bfloat16 v) { return key16(__bfloat16_as_ushort(v), 0x7f80u); }
  static __device__ __forceinline__ __nv_bfloat16 largest(const uint4& v) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
    const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return __hmax(__low2bfloat16(m), __high2bfloat16(m));
  }
  static constexpr uint32_t kLow = 0xff80ff80u, kNone = 0x7fff7fffu;
  static __device__ __forceinline__ void mask(uint4& v, uint32_t bits, uint32_t other) { mask16(v, bits, other); }
};

__device__ __forceinline__ unsigned long long word_of(uint32_t key, uint32_t token) {
  return static_cast<unsigned long long>(key) << 32 | (0xffffffffu - token);
}

template <typename T>
__global__ void __launch_bounds__(kLogitThreads, 2) adjust_logits_kernel(LogitArguments a) {
  using L = Logit<T>;
  constexpr int V = L::kVector, kBlock = kLogitThreads * V;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");   // every CTA runs before another writes to it
  extern __shared__ __align__(16) uint32_t table_s[];   // with a history or biases: keys, counts, bit map, list of slots
  uint32_t* count_s = table_s + a.slots;
  uint32_t* marked_s = count_s + a.slots;
  uint16_t* list_s = reinterpret_cast<uint16_t*>(marked_s + a.widest / 32);
  __shared__ int bias_at_s[kBiases], bias_count_s[kLogitThreads / 32], listed_s;
  __shared__ float bias_s[kBiases];
  __shared__ uint16_t bias_slot_s[kBiases];
  __shared__ unsigned long long part_s[kLogitThreads / 32], slice_s[kRanks];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  uint32_t rank, ranks;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
  const int m = blockIdx.y;
  const T* row = static_cast<const T*>(a.logits) + m * a.logits_stride;
  T* out = static_cast<T*>(a.out) + m * a.out_stride;
  // a place in the row is a token shifted so that places divisible by the vector lie on 16 bytes
  const int shift = int(reinterpret_cast<uintptr_t>(row) % 16 / sizeof(T));
  const bool vectors = reinterpret_cast<uintptr_t>(out) % 16 == reinterpret_cast<uintptr_t>(row) % 16;
  row -= shift;
  out -= shift;
  const int64_t token0 = a.offset - shift;
  const int length = a.tokens ? min(max(a.lengths[m], 0), a.history) : 0;
  const int prompt = a.tokens && a.prompts ? a.prompts[m] : 0;
  const float repetition = a.repetition ? a.repetition[m] : 1.f;
  const float frequency = a.frequency ? a.frequency[m] : 0.f, presence = a.presence ? a.presence[m] : 0.f;
  const uint32_t* mask = reinterpret_cast<const uint32_t*>(a.mask) + m * a.mask_stride;
  const bool tracked = length > 0 || a.biases > 0;
  // Chunks go by the row's own text, whatever the width of its buffer: the whole slice at a time when the table takes all that the row
  // notes, else a block, which has no more tokens than the table takes, with the history read again for each.  (Rows of 300 tokens
  // in a buffer of 32768, chunks by the width of the buffer and by the text: one row 12.8 and 9.0 us, 128 rows 97 and 25, in a
  // buffer of 300 8.2 and 25.  A table of the text's size as well takes 0.5 us off one such row and adds 1 us to 128 rows with texts of
  // 4000.  Texts of 30000: one row 42, 128 rows 373 us.)
  const int noted = length + a.biases;
  const int chunk = noted <= kMost ? a.widest : kBlock;

  // the row's blocks of a piece for each thread go to the CTAs in turn, so that common tokens, which lie together, do not
  // meet in one; a CTA numbers its own places through
  const int end = a.width + shift, turn = __ffs(ranks) - 1;
  auto place_of = [&](int local) { return ((local / kBlock << turn) + int(rank)) * kBlock + local % kBlock; };
  unsigned long long top = 0;                  // of what the list takes
  uint32_t key = 0;                            // of the rest, which it meets in rising order: the largest key,
  uint4 best{};                                // the first piece that has it, and that piece's token
  int64_t token = kNothing;
  auto history = [&](int i) -> int64_t {
    return a.long_tokens ? __ldg(static_cast<const long long*>(a.tokens) + m * a.tokens_stride + i)
                         : __ldg(static_cast<const int*>(a.tokens) + m * a.tokens_stride + i);
  };
  if (tracked) {
    // the slice's logits come to L2 while the history is gathered
    for (int block = threadIdx.x; block * kBlock < a.slice; block += kLogitThreads) {
      const int from = max(place_of(block * kBlock), (shift + V - 1) / V * V), to = min(place_of(block * kBlock) + kBlock, end / V * V);
      if (from < to)
        asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(row + from), "r"(uint32_t((to - from) * sizeof(T))) : "memory");
    }
  }
  for (int base = 0;; base += chunk) {
    const int last = min(base + chunk, a.slice);
    // the chunk's first logits, and their bits of the mask
    uint4 held[kDeep];
    uint64_t bits[kDeep];
    const int first = base + int(threadIdx.x) * V;
    auto load = [&](int i, int local) {
      const int place = place_of(local);
      if (local >= last || place >= end) return;
      if (vectors && place >= shift && place + V <= end) held[i] = *reinterpret_cast<const uint4*>(row + place);
      if (a.mask) {
        const int64_t at = max(token0 + place, int64_t(0)), word = at >> 5;     // a place before the row's first token has no bit
        bits[i] = mask[word];
        if ((at & 31) + V > 32 && word + 1 < a.mask_words) bits[i] |= uint64_t(mask[word + 1]) << 32;
      }
    };
#pragma unroll
    for (int i = 0; i < kDeep; ++i) load(i, first + i * kBlock);
    // the number in the chunk of a token, or none
    auto number = [&](int64_t id) {
      const int64_t place = id - token0;
      if (place < shift || place >= end) return kNoPlace;
      const uint32_t block = uint32_t(place) / kBlock;
      if ((block & (ranks - 1)) != rank) return kNoPlace;
      const uint32_t at = (block >> turn) * kBlock + uint32_t(place) % kBlock - uint32_t(base);
      return at < uint32_t(last - base) ? at : kNoPlace;
    };
    // the table's slot of the token with a number, which it has from now on
    auto slot_of = [&](uint32_t at) {
      uint32_t slot = (at + 1) * 2654435761u >> (__clz(a.slots) + 1);
      for (;;) {
        const uint32_t there = atomicCAS(table_s + slot, 0u, at + 1);
        if (there == 0 || there == at + 1) return slot;
        slot = (slot + 1) & (a.slots - 1);
      }
    };
    // the history's first tokens and the first biases are under way while the table is cleared (a shard of 19 000 with biases
    // 7.5 -> 6.9 us, eight rows of 32 bits 11.6 -> 11.3 us; a short row alone 5.3 -> 5.4 us)
    constexpr int kEarly = 4;
    int64_t early[kEarly];
#pragma unroll
    for (int u = 0; u < kEarly; ++u) early[u] = int(threadIdx.x) + u * kLogitThreads < length ? history(threadIdx.x + u * kLogitThreads) : -1;
    const bool early_entry = int(threadIdx.x) < a.biases;
    const int early_token = early_entry ? a.bias_tokens[m * a.bias_stride + threadIdx.x] : -1;
    const float early_bias = early_entry ? a.bias[m * a.bias_stride + threadIdx.x] : 0.f;
    if (tracked) {
      for (int i = threadIdx.x * 4; i < 2 * a.slots + a.widest / 32; i += kLogitThreads * 4) *reinterpret_cast<uint4*>(table_s + i) = make_uint4(0u, 0u, 0u, 0u);
      if (threadIdx.x == 0) listed_s = 0;
      __syncthreads();
      auto count = [&](int i, int64_t id) {
        const uint32_t at = number(id);
        if (at == kNoPlace) return;
        atomicAdd(count_s + slot_of(at), i >= prompt ? 1u : 0u);
        atomicOr(marked_s + at / 32, 1u << (at % 32));
      };
#pragma unroll
      for (int u = 0; u < kEarly; ++u)
        if (int(threadIdx.x) + u * kLogitThreads < length) count(threadIdx.x + u * kLogitThreads, early[u]);
      int i = threadIdx.x + kEarly * kLogitThreads;
      for (; i + 3 * kLogitThreads < length; i += 4 * kLogitThreads) {
        int64_t ids[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) ids[u] = history(i + u * kLogitThreads);
#pragma unroll
        for (int u = 0; u < 4; ++u) count(i + u * kLogitThreads, ids[u]);
      }
      for (; i < length; i += kLogitThreads) count(i, history(i));
      __syncthreads();
    }
    // the biases of this chunk, in their order
    int biases = 0;
    for (int group = 0; group < a.biases; group += kLogitThreads) {
      const int entry = group + threadIdx.x;
      const uint32_t at = entry < a.biases ? number(group == 0 ? early_token : a.bias_tokens[m * a.bias_stride + entry]) : kNoPlace;
      const bool inside = at != kNoPlace;
      const uint32_t votes = __ballot_sync(0xffffffffu, inside);
      if ((threadIdx.x & 31) == 0) bias_count_s[threadIdx.x >> 5] = __popc(votes);
      __syncthreads();
      int slot = biases + __popc(votes & ((1u << (threadIdx.x & 31)) - 1));
#pragma unroll
      for (int w = 0; w < kLogitThreads / 32; ++w) {
        if (w < int(threadIdx.x >> 5)) slot += bias_count_s[w];
        biases += bias_count_s[w];
      }
      // whether the history has the token: it is in the table before this group's entries come in, and if an entry of a group
      // before brought it, that one's flag says so
      bool seen = false;
      if (inside) {
        uint32_t probe = (at + 1) * 2654435761u >> (__clz(a.slots) + 1);
        while (table_s[probe] != 0 && table_s[probe] != at + 1) probe = (probe + 1) & (a.slots - 1);
        seen = table_s[probe] != 0 && (count_s[probe] & (kBiased | kSeen)) != kBiased;
      }
      __syncthreads();
      if (inside) {
        const uint32_t there = slot_of(at);
        atomicOr(count_s + there, seen ? kBiased | kSeen : kBiased);
        atomicOr(marked_s + at / 32, 1u << (at % 32));
        if (slot < kBiases) {
          bias_slot_s[slot] = uint16_t(there);
          bias_at_s[slot] = int(at);
          bias_s[slot] = group == 0 ? early_bias : a.bias[m * a.bias_stride + entry];
        }
      }
      __syncthreads();
    }
    if (tracked) __syncthreads();
    for (int start = first; start < last; start += kDeep * kBlock) {
#pragma unroll
      for (int i = 0; i < kDeep; ++i) {
        const int local = start + i * kBlock, place = place_of(local);
        if (local >= last || place >= end) break;
        const int64_t id = token0 + place;
        const uint32_t marked = tracked ? marked_s[(local - base) / 32] >> (local % 32) & ((1u << V) - 1) : 0u;
        uint32_t allowed = ~0u;
        if (a.mask) {
          const int64_t at = max(id, int64_t(0));
          allowed = uint32_t(bits[i] >> (at & 31)) << (at - id) | marked;
        }
        uint4 v = held[i];
        const bool whole = vectors && place >= shift && place + V <= end;
        if (whole) {
          load(i, local + kDeep * kBlock);
          if (a.mask) L::mask(v, allowed, L::kLow);
          *reinterpret_cast<uint4*>(out + place) = v;      // marked tokens as they were: the list reads them, here or in `row`
        } else {
          T* values = reinterpret_cast<T*>(&v);
          uint32_t inside = 0;
#pragma unroll
          for (int e = 0; e < V; ++e) inside |= uint32_t(place + e >= shift && place + e < end) << e;
#pragma unroll
          for (int e = 0; e < V; ++e) values[e] = inside >> e & 1u ? row[place + e] : L::narrow(0.f);
          load(i, local + kDeep * kBlock);
          if (a.mask) L::mask(v, allowed, L::kLow);
#pragma unroll
          for (int e = 0; e < V; ++e)
            if (inside >> e & 1u) out[place + e] = values[e];
          L::mask(v, inside, L::kNone);
        }
        if (marked) L::mask(v, ~marked, L::kNone);
        const uint32_t largest = L::key(L::largest(v));
        if (largest > key || token == kNothing) {
          key = largest;
          best = v;
          token = id;
        }
      }
    }
    if (tracked) {
      // the slots in use, listed warp by warp (a shared counter for each new token queued them all)
      int used = 0;
      for (int i = threadIdx.x; i < a.slots; i += kLogitThreads) used += table_s[i] != 0;
      int before = used;
#pragma unroll
      for (int step = 1; step < 32; step <<= 1) {
        const int other = __shfl_up_sync(0xffffffffu, before, step);
        if (int(threadIdx.x & 31) >= step) before += other;
      }
      int to = 0;
      if ((threadIdx.x & 31) == 31) to = atomicAdd(&listed_s, before);
      to = __shfl_sync(0xffffffffu, to, 31) + before - used;
      for (int i = threadIdx.x; i < a.slots; i += kLogitThreads)
        if (table_s[i] != 0) list_s[to++] = uint16_t(i);
      __syncthreads();
      const int listed = listed_s;
      auto finish = [&](int at, uint32_t count, float bias) {
        const int place = place_of(base + at);
        const int64_t id = token0 + place;
        float x = L::widen(row[place]);
        if ((count & (kBiased | kSeen)) != kBiased) {
          x = x > 0.f ? __fdiv_rn(x, repetition) : __fmul_rn(x, repetition);
          x = __fsub_rn(x, __fmul_rn(frequency, float(count & kCount)));
          if (count & kCount) x = __fsub_rn(x, presence);
        }
        if (count & kBiased) x = __fadd_rn(x, bias);
        if (a.mask && !(mask[id >> 5] >> (id & 31) & 1u)) x = -INFINITY;
        const T result = L::narrow(x);
        out[place] = result;
        const unsigned long long word = word_of(L::key(result), uint32_t(id));
        top = word > top ? word : top;
      };
      // the biases of a token are added up in the order of the entries, in 64 bits
      for (int i = threadIdx.x; i < listed; i += kLogitThreads) {
        const int at = int(table_s[list_s[i]]) - 1;
        const uint32_t count = count_s[list_s[i]];
        double sum = 0.0;
        if (count & kBiased) {
          if (biases <= kBiases) continue;      // by the thread of its first entry, below
          for (int e = 0; e < a.biases; ++e)
            if (number(a.bias_tokens[m * a.bias_stride + e]) == uint32_t(at)) sum += a.bias[m * a.bias_stride + e];
        }
        finish(at, count, float(sum));
      }
      for (int i = threadIdx.x; i < biases && biases <= kBiases; i += kLogitThreads) {
        const int at = bias_at_s[i];
        double sum = 0.0;
        bool first_entry = true;
        for (int e = 0; e < biases; ++e) {
          if (bias_at_s[e] != at) continue;
          first_entry = first_entry && e >= i;
          sum += bias_s[e];
        }
        if (first_entry) finish(at, count_s[bias_slot_s[i]], float(sum));
      }
    }
    if (last == a.slice) break;
    __syncthreads();
  }
  if (token != kNothing) {
    const T* values = reinterpret_cast<const T*>(&best);
    int first = V - 1;
#pragma unroll
    for (int e = V - 1; e >= 0; --e)
      if (L::key(values[e]) == key) first = e;
    // (nothing but NaN, and what is no token, in a piece: its first token)
    const unsigned long long word = word_of(key, uint32_t(max(token + first, a.offset)));
    top = word > top ? word : top;
  }
#pragma unroll
  for (int step = 16; step; step >>= 1) {
    const unsigned long long other = __shfl_xor_sync(0xffffffffu, top, step);
    top = other > top ? other : top;
  }
  if ((threadIdx.x & 31) == 0) part_s[threadIdx.x >> 5] = top;
  __syncthreads();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (threadIdx.x < 32) {
    top = threadIdx.x < kLogitThreads / 32 ? part_s[threadIdx.x] : 0;
#pragma unroll
    for (int step = kLogitThreads / 64; step; step >>= 1) {
      const unsigned long long other = __shfl_xor_sync(0xffffffffu, top, step);
      top = other > top ? other : top;
    }
    if (threadIdx.x == 0) {
      uint32_t local = uint32_t(__cvta_generic_to_shared(&slice_s[rank])), remote;
      asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(remote) : "r"(local));
      asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(remote), "l"(top) : "memory");
    }
  }
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (rank == 0 && threadIdx.x == 0) {
    for (uint32_t r = 0; r < ranks; ++r) top = slice_s[r] > top ? slice_s[r] : top;
    if (a.best) a.best[m] = top;
    if (a.picked) a.picked[m] = 0xffffffffu - uint32_t(top);
  }
}

// Dynamic shared memory of a launch with tables of `slots` and chunks of up to `widest` tokens.
size_t table_bytes(int slots, int widest) { return size_t(slots) * 8 + slots * 3 / 4 * 2 + widest / 8; }

template <typename T>
int launch_logits(LogitArguments& a, int M, void* stream) {
  int device = 0;
  cudaGetDevice(&device);
  static std::atomic<uint64_t> opted{0};
  if (!(opted.load(std::memory_order_acquire) >> (device & 63) & 1)) {
    cudaError_t set = cudaFuncSetAttribute(adjust_logits_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, device_info().max_smem_optin - 8192);
    if (set == cudaSuccess) set = cudaFuncSetAttribute(adjust_logits_kernel<T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (set != cudaSuccess) return cuda_fail(set, "adjust_logits attributes");
    opted.fetch_or(uint64_t(1) << (device & 63), std::memory_order_release);
  }
  cudaLaunchConfig_t config{};
  config.blockDim = dim3(kLogitThreads);
  config.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attribute[2];
  attribute[0].id = cudaLaunchAttributeClusterDimension;
  attribute[0].val.clusterDim.y = attribute[0].val.clusterDim.z = 1;
  attribute[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute[1].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attribute;
  constexpr int kBlock = kLogitThreads * Logit<T>::kVector;
  const bool tracked = a.tokens || a.bias;
  // a CTA's places: as many blocks of a piece for each thread as the longest of them has; the bit map of a chunk has 64 KB at
  // most, and the table room for what the widest text that fits the buffer needs
  auto shape = [&](int ranks) {
    const int blocks = (a.width + 7 + kBlock - 1) / kBlock;
    a.slice = (blocks + ranks - 1) / ranks * kBlock;
    a.widest = a.slice < 1 << 19 ? a.slice : 1 << 19;
    config.gridDim = dim3(ranks, M);
    config.dynamicSmemBytes = tracked ? table_bytes(a.slots, a.widest) : 0;
    attribute[0].val.clusterDim.x = ranks;
  };
  // CTAs of a row: up to sixteen, of 4096 tokens or more, and in all no more than run at once, which for clusters is less than
  // for CTAs, since a cluster lies within a group of SMs (of sixteen 14 run at once, 224 of 296 CTAs): 16 rows of 50257 in 32 bits
  // took two turns of clusters of sixteen, 15 us, and take one of clusters of eight, 11.  The answer for the last call's sizes is kept: asking the runtime takes some microseconds.
  thread_local struct { int device, rows, width, slots; bool tracked; int ranks; } last{-1, 0, 0, 0, false, 0};
  if (last.device != device || last.rows != M || last.width != a.width || last.slots != a.slots || last.tracked != tracked) {
    int ranks = 1;
    for (int next = 2; next <= kRanks && next / 2 * 4096 < a.width; next *= 2) {
      shape(next);
      config.numAttrs = 1;
      int clusters = 0;
      const cudaError_t asked = cudaOccupancyMaxActiveClusters(&clusters, adjust_logits_kernel<T>, &config);
      if (asked != cudaSuccess) return cuda_fail(asked, "adjust_logits clusters");
      if (clusters < M) break;
      ranks = next;
    }
    last = {device, M, a.width, a.slots, tracked, ranks};
  }
  shape(last.ranks);
  config.numAttrs = 2;
  const cudaError_t launched = cudaLaunchKernelEx(&config, adjust_logits_kernel<T>, a);
  if (launched != cudaSuccess) return cuda_fail(launched, "adjust_logits launch");
  return MKB_OK;
}

}  // namespace
}  // namespace mkb

extern "C" int mkb_adjust_logits(const void* logits, void* out, const void* tokens, const int* lengths, const int* prompts,
                                 const float* repetition, const float* frequency, const float* presence, const int* bias_tokens,
                                 const float* bias, const int* mask, void* best, void* picked, int M, int64_t width,
                                 int64_t logits_stride, int64_t out_stride, int64_t history, int64_t tokens_stride, int64_t biases,
                                 int64_t bias_stride, int64_t mask_words, int64_t mask_stride, int64_t offset, int long_tokens,
                                 int dtype, void* stream) {
  using namespace mkb;
  MKB_REQUIRE(M >= 0 && width >= 1 && logits_stride >= 0 && out_stride >= 0 && history >= 0 && biases >= 0 && offset >= 0 &&
                  width < (int64_t(1) << 30) && offset + width < (int64_t(1) << 31) && history < (int64_t(1) << 30) &&
                  biases < (int64_t(1) << 30),
              MKB_E_ARGUMENT, "adjust_logits: bad shape");
  MKB_REQUIRE(M <= 65535, MKB_E_UNSUPPORTED, "adjust_logits: %d rows", M);
  if (M == 0) return MKB_OK;
  MKB_REQUIRE(logits && out, MKB_E_ARGUMENT, "adjust_logits: null pointer");
  MKB_REQUIRE(M == 1 || out_stride >= width, MKB_E_ARGUMENT, "adjust_logits: rows of the output overlap");
  const int64_t size = dtype_bytes(dtype);
  // side by side in the rows of one buffer
  const int64_t pitch = logits_stride * size, apart = int64_t(reinterpret_cast<uintptr_t>(out) - reinterpret_cast<uintptr_t>(logits));
  const int64_t beside = pitch > 0 ? (apart % pitch + pitch) % pitch : 0;
  MKB_REQUIRE((logits == out && (M == 1 || logits_stride == out_stride)) ||
                  (logits_stride == out_stride && beside >= width * size && pitch - beside >= width * size) ||
                  !overlap(logits, ((M - 1) * logits_stride + width) * size, out, ((M - 1) * out_stride + width) * size),
              MKB_E_ARGUMENT, "adjust_logits: the output overlaps the logits");
  MKB_REQUIRE(!tokens || history == 0 || lengths, MKB_E_ARGUMENT, "adjust_logits: a history needs its lengths");
  MKB_REQUIRE((bias_tokens != nullptr) == (bias != nullptr), MKB_E_ARGUMENT, "adjust_logits: biases need tokens and values");
  MKB_REQUIRE(!mask || (mask_words << 5) >= offset + width, MKB_E_ARGUMENT, "adjust_logits: a mask of %lld words ends before token %lld",
              (long long)mask_words, (long long)(offset + width));
  LogitArguments a{logits, out, history ? tokens : nullptr, lengths, prompts, repetition, frequency, presence, bias_tokens, bias, mask,
                   static_cast<unsigned long long*>(best), static_cast<long long*>(picked), logits_stride, out_stride, tokens_stride,
                   bias_stride, mask_words, mask_stride, offset, int(width), int(history), bias ? int(biases) : 0, long_tokens, 0, 0, 0};
  const int64_t noted = (a.tokens ? history : 0) + a.biases;
  a.slots = kLogitThreads;
  while (a.slots < kSlots && a.slots * 3 / 4 < noted) a.slots *= 2;
  static_assert(kMost == kSlots * 3 / 4, "the table's size");
  static_assert(kLogitThreads * 8 <= kMost, "a block fits the table");
  switch (dtype) {
    case MKB_F16: return launch_logits<__half>(a, M, stream);
    case MKB_BF16: return launch_logits<__nv_bfloat16>(a, M, stream);
    case MKB_F32: return launch_logits<float>(a, M, stream);
    default: break;
  }
  set_error("adjust_logits: dtype tag %d (fp16, bf16 and fp32 supported)", dtype);
  return MKB_E_UNSUPPORTED;
}
