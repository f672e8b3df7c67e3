// Penalties for repeated tokens, biases and a grammar's mask on the logits of a decode step, with the greedy pick.
// For token v of a row, x its logit, r / f / p the row's penalties:
//   v in the history:                 x = x > 0 ? x / r : x * r
//   c times in what was generated:    x = x - f * c,  and x = x - p when c > 0
//   biases b of v:                    x = x + sum b
//   the mask's bit is 0:              x = -inf
// in fp32 in this order, rounded once to the logits' type.
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
  int64_t logits_stride, out_stride, tokens_stride, bias_stride, mask_stride, offset;
  int width, history, biases, long_tokens, slice;
};

constexpr int kLogitThreads = 512;
constexpr int kChunk = 8192;             // tokens whose counts lie in shared memory at a time
constexpr uint32_t kSeen = 0x80000000u;  // the high bit of a count: the token is in the history

// fp16 keeps the 16-bit keys of the arg-max kernel, so that their words compare; NaN ranks lowest, ties go to the lower token.
__device__ __forceinline__ uint32_t sortable(float v, int) {
  const uint32_t bits = __float_as_uint(v);
  if ((bits & 0x7fffffffu) > 0x7f800000u) return 0u;
  return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}
__device__ __forceinline__ uint32_t sortable(unsigned short bits, int infinity) {
  if ((bits & 0x7fffu) > infinity) return 0u;
  return bits & 0x8000u ? ~uint32_t(bits) & 0xffffu : bits | 0x8000u;
}
__device__ __forceinline__ uint32_t key_of(__half v) { return sortable(__half_as_ushort(v), 0x7c00); }
__device__ __forceinline__ uint32_t key_of(__nv_bfloat16 v) { return sortable(__bfloat16_as_ushort(v), 0x7f80); }
__device__ __forceinline__ uint32_t key_of(float v) { return sortable(v, 0); }

template <typename T> __device__ __forceinline__ T rounded(float v);
template <> __device__ __forceinline__ __half rounded(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 rounded(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ float rounded(float v) { return v; }
__device__ __forceinline__ float widened(__half v) { return __half2float(v); }
__device__ __forceinline__ float widened(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float widened(float v) { return v; }

// A cluster per row, a CTA per slice of the vocabulary: counts of the slice's tokens are gathered in shared memory from the
// whole history, the slice is adjusted, and the CTAs' best words meet in the first one's shared memory.
template <typename T>
__global__ void __launch_bounds__(kLogitThreads) adjust_logits_kernel(LogitArguments a) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");   // every CTA runs before another writes to it
  asm volatile("griddepcontrol.wait;" ::: "memory");
  __shared__ uint32_t count_s[kChunk];
  __shared__ unsigned long long part_s[kLogitThreads / 32], slice_s[16];
  uint32_t rank, ranks;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
  const int m = blockIdx.y;
  const T* row = static_cast<const T*>(a.logits) + m * a.logits_stride;
  T* out = static_cast<T*>(a.out) + m * a.out_stride;
  const int length = a.tokens ? min(max(a.lengths[m], 0), a.history) : 0;
  const int prompt = a.tokens && a.prompts ? a.prompts[m] : 0;
  const float repetition = a.repetition ? a.repetition[m] : 1.f;
  const float frequency = a.frequency ? a.frequency[m] : 0.f, presence = a.presence ? a.presence[m] : 0.f;
  unsigned long long top = 0;
  const int begin = int(rank) * a.slice, end = min(begin + a.slice, a.width);
  for (int base = begin; base < end; base += kChunk) {
    const int size = min(kChunk, end - base);
    const int64_t token0 = a.offset + base;
    if (length > 0) {
      for (int i = threadIdx.x; i < size; i += kLogitThreads) count_s[i] = 0;
      __syncthreads();
      for (int i = threadIdx.x; i < length; i += kLogitThreads) {
        const int64_t token = a.long_tokens ? static_cast<const long long*>(a.tokens)[m * a.tokens_stride + i]
                                            : static_cast<const int*>(a.tokens)[m * a.tokens_stride + i];
        const int64_t at = token - token0;
        if (at >= 0 && at < size) {
          if (i >= prompt) atomicAdd(&count_s[at], 1u);
          atomicOr(&count_s[at], kSeen);
        }
      }
      __syncthreads();
    }
    for (int i = threadIdx.x; i < size; i += kLogitThreads) {
      float x = widened(row[base + i]);
      if (length > 0) {
        const uint32_t count = count_s[i];
        if (count) {
          x = x > 0.f ? __fdiv_rn(x, repetition) : __fmul_rn(x, repetition);
          x = __fsub_rn(x, __fmul_rn(frequency, float(count & ~kSeen)));
          if (count & ~kSeen) x = __fsub_rn(x, presence);
        }
      }
      if (a.biases) {
        double sum = 0.0;
        bool any = false;
        for (int e = 0; e < a.biases; ++e)
          if (a.bias_tokens[m * a.bias_stride + e] == token0 + i) { sum += a.bias[m * a.bias_stride + e]; any = true; }
        if (any) x = __fadd_rn(x, float(sum));
      }
      if (a.mask) {
        const int64_t token = token0 + i;
        if (!(uint32_t(a.mask[m * a.mask_stride + (token >> 5)]) >> (token & 31) & 1u)) x = -INFINITY;
      }
      const T result = rounded<T>(x);
      out[base + i] = result;
      const unsigned long long candidate = static_cast<unsigned long long>(key_of(result)) << 32 | (0xffffffffu - uint32_t(token0 + i));
      top = candidate > top ? candidate : top;
    }
    __syncthreads();
  }
#pragma unroll
  for (int step = 16; step; step >>= 1) {
    const unsigned long long other = __shfl_xor_sync(0xffffffffu, top, step);
    top = other > top ? other : top;
  }
  if ((threadIdx.x & 31) == 0) part_s[threadIdx.x >> 5] = top;
  __syncthreads();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (threadIdx.x == 0) {
    for (int w = 1; w < kLogitThreads / 32; ++w) top = part_s[w] > top ? part_s[w] : top;
    uint32_t local = uint32_t(__cvta_generic_to_shared(&slice_s[rank])), remote;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(remote) : "r"(local));
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(remote), "l"(top) : "memory");
  }
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (rank == 0 && threadIdx.x == 0) {
    for (uint32_t r = 0; r < ranks; ++r) top = slice_s[r] > top ? slice_s[r] : top;
    if (a.best) a.best[m] = top;
    if (a.picked) a.picked[m] = 0xffffffffu - uint32_t(top);
  }
}

template <typename T>
int launch_logits(const LogitArguments& a, int M, int ranks, void* stream) {
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(ranks, M);
  config.blockDim = dim3(kLogitThreads);
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
                   bias_stride, mask_stride, offset, int(width), int(history), bias ? int(biases) : 0, long_tokens, 0};
  const int ranks = 8;
  a.slice = int((width + ranks - 1) / ranks);
  switch (dtype) {
    case MKB_F16: return launch_logits<__half>(a, M, ranks, stream);
    case MKB_BF16: return launch_logits<__nv_bfloat16>(a, M, ranks, stream);
    case MKB_F32: return launch_logits<float>(a, M, ranks, stream);
    default: break;
  }
  set_error("adjust_logits: dtype tag %d (fp16, bf16 and fp32 supported)", dtype);
  return MKB_E_UNSUPPORTED;
}
