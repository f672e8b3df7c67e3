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
  int width, history, biases, long_tokens, slice, chunk;
};

// What bounds it: for many rows the logits, read and written once (4 bytes a token in 16 bits); for few, the chain of
// launch, history and one reduction.  So a row is spread over a cluster of CTAs, as many as keep the GPU busy, each with a
// slice of the vocabulary.  A CTA reads the whole history once, gathers the slice's tokens with their counts in a hash table
// in shared memory (no [rows, vocabulary] state exists anywhere) and marks them in a bit map, while its first logits are
// under way.  Then the slice passes in 16-byte pieces as it is, masked in its own type, but for the marked tokens, and the
// greedy pick looks at a piece's maximum only; the marked tokens follow from the table's list, one a thread.  The CTAs' best
// words meet in the first one's shared memory, since an order of (value, lower token) does not depend on who comes first.
// Tried for 128 rows of 128256 tokens with 4000 in the history, 300 biases and a mask: penalties worked out where a piece
// met them 115 us (almost every warp did all of it for all of its tokens), a count per token in shared memory, chunk by chunk,
// 77 us, counts of the history's shares added into the other CTAs' memory 96 us (common tokens queued there).
constexpr int kLogitThreads = 512;
constexpr int kDeep = 4;                  // pieces of a thread under way
constexpr int kSlots = 8192;              // of the hash table
constexpr int kMost = 6144;               // tokens it takes; more history than that goes by chunks of that many tokens
constexpr int kRanks = 16;                // CTAs of a row, at most
constexpr uint32_t kSeen = 0x80000000u;   // of a count: the token is in the prompt
constexpr uint32_t kBiased = 0x40000000u; // of a count: the token has a bias
constexpr uint32_t kCount = kBiased - 1;  // how often it was generated
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
  static __device__ __forceinline__ void mask(uint4& v, uint32_t bits) {
    v.x = bits & 1u ? v.x : 0xff800000u; v.y = bits & 2u ? v.y : 0xff800000u;
    v.z = bits & 4u ? v.z : 0xff800000u; v.w = bits & 8u ? v.w : 0xff800000u;
  }
};
// fp16 and bf16: the 16-bit keys of the arg-max kernel, so that their words compare.
__device__ __forceinline__ uint32_t key16(uint32_t bits, uint32_t infinity) {
  if ((bits & 0x7fffu) > infinity) return 0u;
  if (bits == 0x8000u) return 0x8000u;
  return bits & 0x8000u ? ~bits & 0xffffu : bits | 0x8000u;
}
__device__ __forceinline__ uint32_t mask16(uint32_t pair, uint32_t bits, uint32_t infinity) {
  const uint32_t keep = (bits & 1u ? 0xffffu : 0u) | (bits & 2u ? 0xffff0000u : 0u);
  return (pair & keep) | (infinity & ~keep);
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
  static __device__ __forceinline__ void mask(uint4& v, uint32_t bits) {
    v.x = mask16(v.x, bits, 0xfc00fc00u); v.y = mask16(v.y, bits >> 2, 0xfc00fc00u);
    v.z = mask16(v.z, bits >> 4, 0xfc00fc00u); v.w = mask16(v.w, bits >> 6, 0xfc00fc00u);
  }
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
  static __device__ __forceinline__ void mask(uint4& v, uint32_t bits) {
    v.x = mask16(v.x, bits, 0xff80ff80u); v.y = mask16(v.y, bits >> 2, 0xff80ff80u);
    v.z = mask16(v.z, bits >> 4, 0xff80ff80u); v.w = mask16(v.w, bits >> 6, 0xff80ff80u);
  }
};

__device__ __forceinline__ unsigned long long word_of(uint32_t key, uint32_t token) {
  return static_cast<unsigned long long>(key) << 32 | (0xffffffffu - token);
}

template <typename T>
__global__ void __launch_bounds__(kLogitThreads, 2) adjust_logits_kernel(LogitArguments a) {
  using L = Logit<T>;
  constexpr int V = L::kVector;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");   // every CTA runs before another writes to it
  extern __shared__ __align__(16) uint32_t table_s[];   // with a history or biases: keys, counts, bit map, list of slots
  uint32_t* count_s = table_s + kSlots;
  uint32_t* marked_s = count_s + kSlots;
  uint16_t* list_s = reinterpret_cast<uint16_t*>(marked_s + a.chunk / 32);
  __shared__ int bias_at_s[kBiases], bias_count_s[kLogitThreads / 32], listed_s;
  __shared__ float bias_s[kBiases];
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

  const int begin = max(int(rank) * a.slice, shift), end = min(int(rank + 1) * a.slice, a.width + shift);
  unsigned long long top = 0;                  // of what the list takes
  uint32_t key = 0, token = 0;                 // of the rest, which it meets in rising order
  bool any = false;
  auto history = [&](int i) -> int64_t {
    return a.long_tokens ? __ldg(static_cast<const long long*>(a.tokens) + m * a.tokens_stride + i)
                         : __ldg(static_cast<const int*>(a.tokens) + m * a.tokens_stride + i);
  };
  for (int base = int(rank) * a.slice;; base += a.chunk) {
    const int low = max(base, begin), high = min(base + a.chunk, end);
    const int64_t first = token0 + base;      // token of the chunk's first place
    // the chunk's first logits, and their bits of the mask
    uint4 held[kDeep];
    uint64_t bits[kDeep];
    const int place0 = base + int(threadIdx.x) * V;
    auto load = [&](int i, int place) {
      if (place >= high) return;
      if (vectors && place >= low && place + V <= high) held[i] = *reinterpret_cast<const uint4*>(row + place);
      if (a.mask) {
        const int64_t at = max(token0 + place, int64_t(0)), word = at >> 5;     // a place before the row's first token has no bit
        bits[i] = mask[word];
        if ((at & 31) + V > 32 && word + 1 < a.mask_words) bits[i] |= uint64_t(mask[word + 1]) << 32;
      }
    };
#pragma unroll
    for (int i = 0; i < kDeep; ++i) load(i, place0 + i * kLogitThreads * V);
    // counts `add` for, or flags, the token at a place of the chunk
    auto note = [&](uint32_t at, uint32_t add, uint32_t flag) {
      uint32_t slot = (at + 1) * 2654435761u >> 19;
      static_assert(kSlots == 1 << 13, "the hash leaves 13 bits");
      for (;; slot = (slot + 1) % kSlots) {
        uint32_t key_there = *static_cast<volatile uint32_t*>(table_s + slot);
        if (key_there == 0) {
          key_there = atomicCAS(table_s + slot, 0u, at + 1);
          if (key_there == 0) {
            list_s[atomicAdd(&listed_s, 1)] = uint16_t(slot);
            atomicOr(marked_s + at / 32, 1u << (at % 32));
            break;
          }
        }
        if (key_there == at + 1) break;
      }
      if (flag) atomicOr(count_s + slot, flag);
      else atomicAdd(count_s + slot, add);
    };
    if (tracked) {
      for (int i = threadIdx.x * 4; i < 2 * kSlots + a.chunk / 32; i += kLogitThreads * 4) *reinterpret_cast<uint4*>(table_s + i) = make_uint4(0u, 0u, 0u, 0u);
      if (threadIdx.x == 0) listed_s = 0;
      __syncthreads();
      const int64_t from = first + (low - base);
      const uint32_t size = uint32_t(high - low);
      auto count = [&](int i, int64_t id) {
        if (uint64_t(id - from) < size) note(uint32_t(id - first), 1u, i >= prompt ? 0u : kSeen);
      };
      int i = threadIdx.x;
      for (; i + 3 * kLogitThreads < length; i += 4 * kLogitThreads) {
        int64_t ids[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) ids[u] = history(i + u * kLogitThreads);
#pragma unroll 1
        for (int u = 0; u < 4; ++u) count(i + u * kLogitThreads, u == 0 ? ids[0] : u == 1 ? ids[1] : u == 2 ? ids[2] : ids[3]);
      }
      for (; i < length; i += kLogitThreads) count(i, history(i));
    }
    // the biases of this chunk, in their order
    int biases = 0;
    for (int group = 0; group < a.biases; group += kLogitThreads) {
      const int entry = group + threadIdx.x;
      const int64_t id = entry < a.biases ? a.bias_tokens[m * a.bias_stride + entry] : -1, at = id - first;
      const bool inside = id >= 0 && at >= low - base && at < high - base;
      const uint32_t votes = __ballot_sync(0xffffffffu, inside);
      if ((threadIdx.x & 31) == 0) bias_count_s[threadIdx.x >> 5] = __popc(votes);
      __syncthreads();
      int slot = biases + __popc(votes & ((1u << (threadIdx.x & 31)) - 1));
#pragma unroll
      for (int w = 0; w < kLogitThreads / 32; ++w) {
        if (w < int(threadIdx.x >> 5)) slot += bias_count_s[w];
        biases += bias_count_s[w];
      }
      if (inside) {
        note(uint32_t(at), 0u, kBiased);
        if (slot < kBiases) {
          bias_at_s[slot] = int(at);
          bias_s[slot] = a.bias[m * a.bias_stride + entry];
        }
      }
      __syncthreads();
    }
    if (tracked) __syncthreads();
    for (int start = place0; start < high; start += kDeep * kLogitThreads * V) {
#pragma unroll
      for (int i = 0; i < kDeep; ++i) {
        const int place = start + i * kLogitThreads * V, local = place - base;
        if (place >= high) break;
        const int64_t id = token0 + place;
        if (!any) token = uint32_t(token0 + max(place, low));     // a row of NaN gives its first token
        any = true;
        const bool whole = place >= low && place + V <= high;
        uint4 v = held[i];
        T* values = reinterpret_cast<T*>(&v);
        if (!(vectors && whole)) {
#pragma unroll
          for (int e = 0; e < V; ++e) values[e] = place + e >= low && place + e < high ? row[place + e] : L::narrow(-INFINITY);
        }
        if (a.mask) {
          const int64_t at = max(id, int64_t(0));
          L::mask(v, uint32_t(bits[i] >> (at & 31)) << (at - id));
        }
        load(i, place + kDeep * kLogitThreads * V);
        const uint32_t marked = tracked ? marked_s[local / 32] >> (local % 32) & ((1u << V) - 1) : 0u;
        if (vectors && whole && marked == 0) {
          *reinterpret_cast<uint4*>(out + place) = v;
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e) {
            if (place + e >= low && place + e < high && !(marked >> e & 1u)) out[place + e] = values[e];
            else values[e] = L::narrow(__int_as_float(0x7fffffff));      // none, or one of the list
          }
        }
        const uint32_t largest = L::key(L::largest(v));
        if (largest > key) {
          key = largest;
#pragma unroll
          for (int e = V - 1; e >= 0; --e)
            if (L::key(values[e]) == largest) token = uint32_t(id + e);
        }
      }
    }
    if (tracked) {
      __syncthreads();
      const int listed = listed_s;
      for (int i = threadIdx.x; i < listed; i += kLogitThreads) {
        const int at = int(table_s[list_s[i]]) - 1;
        const uint32_t count = count_s[list_s[i]];
        const int64_t id = first + at;
        float x = L::widen(row[base + at]);
        if (count & (kSeen | kCount)) {
          x = x > 0.f ? __fdiv_rn(x, repetition) : __fmul_rn(x, repetition);
          x = __fsub_rn(x, __fmul_rn(frequency, float(count & kCount)));
          if (count & kCount) x = __fsub_rn(x, presence);
        }
        if (count & kBiased) {      // added up in the order of the entries, in 64 bits
          double sum = 0.0;
          if (biases <= kBiases) {
            for (int e = 0; e < biases; ++e) sum += bias_at_s[e] == at ? double(bias_s[e]) : 0.0;
          } else {
            for (int e = 0; e < a.biases; ++e) sum += a.bias_tokens[m * a.bias_stride + e] == id ? double(a.bias[m * a.bias_stride + e]) : 0.0;
          }
          x = __fadd_rn(x, float(sum));
        }
        if (a.mask && !(mask[id >> 5] >> (id & 31) & 1u)) x = -INFINITY;
        const T result = L::narrow(x);
        out[base + at] = result;
        const unsigned long long word = word_of(L::key(result), uint32_t(id));
        top = word > top ? word : top;
      }
    }
    if (base + a.chunk >= end) break;
    __syncthreads();
  }
  if (any) {
    const unsigned long long word = word_of(key, token);
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

constexpr int kTableBytes = kSlots * 8 + kMost * 2;

template <typename T>
int launch_logits(const LogitArguments& a, int M, int ranks, void* stream) {
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(ranks, M);
  config.blockDim = dim3(kLogitThreads);
  config.dynamicSmemBytes = a.tokens || a.bias ? kTableBytes + a.chunk / 8 : 0;
  int device = 0;
  cudaGetDevice(&device);
  static std::atomic<uint64_t> opted{0};
  if (!(opted.load(std::memory_order_acquire) >> (device & 63) & 1)) {
    cudaError_t set = cudaFuncSetAttribute(adjust_logits_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, device_info().max_smem_optin - 8192);
    if (set == cudaSuccess) set = cudaFuncSetAttribute(adjust_logits_kernel<T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (set != cudaSuccess) return cuda_fail(set, "adjust_logits attributes");
    opted.fetch_or(uint64_t(1) << (device & 63), std::memory_order_release);
  }
  config.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attribute[2];
  attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute[0].val.programmaticStreamSerializationAllowed = 1;
  attribute[1].id = cudaLaunchAttributeClusterDimension;
  attribute[1].val.clusterDim.x = ranks;
  attribute[1].val.clusterDim.y = attribute[1].val.clusterDim.z = 1;
  config.attrs = attribute;
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
  MKB_REQUIRE(!tokens || history == 0 || lengths, MKB_E_ARGUMENT, "adjust_logits: a history needs its lengths");
  MKB_REQUIRE((bias_tokens != nullptr) == (bias != nullptr), MKB_E_ARGUMENT, "adjust_logits: biases need tokens and values");
  MKB_REQUIRE(!mask || (mask_words << 5) >= offset + width, MKB_E_ARGUMENT, "adjust_logits: a mask of %lld words ends before token %lld",
              (long long)mask_words, (long long)(offset + width));
  LogitArguments a{logits, out, history ? tokens : nullptr, lengths, prompts, repetition, frequency, presence, bias_tokens, bias, mask,
                   static_cast<unsigned long long*>(best), static_cast<long long*>(picked), logits_stride, out_stride, tokens_stride,
                   bias_stride, mask_words, mask_stride, offset, int(width), int(history), bias ? int(biases) : 0, long_tokens, 0, 0};
  // CTAs of a row: up to sixteen, of 4096 tokens or more (one piece a thread), and two an SM in all
  int ranks = 1;
  while (ranks < kRanks && int64_t(ranks) * 4096 < width && int64_t(ranks) * M <= device_info().sm_count) ranks *= 2;
  a.slice = int((width + 7 + ranks - 1) / ranks + 127) / 128 * 128;
  // a chunk holds no more tokens of a history than the table takes, and its bit map is 64 KB at most
  a.chunk = (a.tokens ? history : 0) + a.biases <= kMost ? (a.slice < 1 << 19 ? a.slice : 1 << 19) : kMost;
  switch (dtype) {
    case MKB_F16: return launch_logits<__half>(a, M, ranks, stream);
    case MKB_BF16: return launch_logits<__nv_bfloat16>(a, M, ranks, stream);
    case MKB_F32: return launch_logits<float>(a, M, ranks, stream);
    default: break;
  }
  set_error("adjust_logits: dtype tag %d (fp16, bf16 and fp32 supported)", dtype);
  return MKB_E_UNSUPPORTED;
}
