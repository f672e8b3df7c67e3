// Attention of one new token per sequence over a paged key-value cache.
//   s[h, p] = scale * q[h] . k[p],   w[h, p] = exp(s[h, p] - max) / sum,   out[h] = sum_p w[h, p] v[p]
// with the query heads h of a group sharing one key-value head; optionally acc[p] += sum over the group of w[h, p].
#include "paged.cuh"

namespace mkb {
namespace {

__device__ unsigned int g_paged_attention_status = 0;

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int offset = 16; offset; offset >>= 1) v += __shfl_xor_sync(0xffffffffu, v, offset);
  return v;
}

struct AttentionArguments {
  PagedLayout layout;
  const void* q;
  const int* positions;
  const int* lengths;
  void* k_pages;
  void* v_pages;
  void* out;
  float* weights;
  int64_t q_row, q_head;    // strides in elements
  int q_heads, kv_heads, rope;
  float theta, scale;
};

// cos and sin of position * theta^(-i / half): the angle in 64 bits, since a far position times a frequency rounded to 32
// bits is off by hundredths of a turn, then reduced to a turn.
__device__ __forceinline__ void rotation(int position, int i, int half, float theta, float& cosine, float& sine) {
  const double turns = double(position) * exp2(-log2(double(theta)) * double(i) / double(half)) * 0.15915494309189533577;
  sincospif(2.f * float(turns - rint(turns)), &sine, &cosine);
}

template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }

// One CTA per (key-value head, sequence); a warp takes slots, its lanes the dimensions.
constexpr int kSimpleWarps = 8;

template <typename T, int D>
__global__ void __launch_bounds__(kSimpleWarps * 32) paged_attention_simple_kernel(AttentionArguments a) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  constexpr int L = D / 32;
  __shared__ float q_s[D], acc_s[kSimpleWarps][D], max_s[kSimpleWarps], sum_s[kSimpleWarps];
  extern __shared__ float norm_s[];   // [group][2]
  const int kv = blockIdx.x, m = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = a.q_heads / a.kv_heads, capacity = a.layout.capacity();
  const int* table = a.layout.tables + m * a.layout.table_stride;
  const T* source = static_cast<const T*>(a.q) + m * a.q_row;
  int length = a.lengths[m];
  const bool idle = length < 0;
  if (length > capacity - a.rope) {
    if (threadIdx.x == 0) atomicOr(&g_paged_attention_status, 1u);
    length = capacity;
  } else if (a.rope && !idle) {
    const uint32_t at = a.layout.vector_of(table, kv, length);
    if (at == kNoSlot) {
      if (threadIdx.x == 0) atomicOr(&g_paged_attention_status, 1u);
    } else {
      const T* k = source + int64_t(a.q_heads + kv) * D;
      const T* v = k + int64_t(a.kv_heads) * D;
      for (int i = threadIdx.x; i < D / 2; i += blockDim.x) {
        float cosine, sine;
        rotation(a.positions[m], i, D / 2, a.theta, cosine, sine);
        const float lo = to_float(k[i]), hi = to_float(k[i + D / 2]);
        static_cast<T*>(a.k_pages)[int64_t(at) * 8 + i] = from_float<T>(lo * cosine - hi * sine);
        static_cast<T*>(a.k_pages)[int64_t(at) * 8 + i + D / 2] = from_float<T>(hi * cosine + lo * sine);
      }
      for (int i = threadIdx.x; i < D; i += blockDim.x) static_cast<T*>(a.v_pages)[int64_t(at) * 8 + i] = v[i];
      if (a.weights != nullptr && threadIdx.x == 0) a.weights[a.layout.weight_of(table, a.kv_heads, kv, length)] = 0.f;
    }
    ++length;
  }
  auto load_query = [&](int head) {
    __syncthreads();
    const T* q = source + int64_t(head) * a.q_head;
    for (int i = threadIdx.x; i < D / 2; i += blockDim.x) {
      float lo = to_float(q[i]), hi = to_float(q[i + D / 2]), cosine = 1.f, sine = 0.f;
      if (a.rope) rotation(a.positions[m], i, D / 2, a.theta, cosine, sine);
      q_s[i] = (lo * cosine - hi * sine) * a.scale;
      q_s[i + D / 2] = (hi * cosine + lo * sine) * a.scale;
    }
    __syncthreads();
  };
  auto score = [&](int p, uint32_t& at) {
    at = a.layout.vector_of(table, kv, p);
    if (at == kNoSlot) {
      if (lane == 0) atomicOr(&g_paged_attention_status, 1u);
      return -INFINITY;
    }
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < L; ++i) dot += q_s[i * 32 + lane] * to_float(static_cast<const T*>(a.k_pages)[int64_t(at) * 8 + i * 32 + lane]);
    return warp_sum(dot);
  };
  for (int g = 0; g < group; ++g) {
    const int head = kv * group + g;
    load_query(head);
    float top = -INFINITY, sum = 0.f, acc[L];
#pragma unroll
    for (int i = 0; i < L; ++i) acc[i] = 0.f;
    for (int p = warp; p < length; p += kSimpleWarps) {
      uint32_t at;
      const float s = score(p, at);
      if (at == kNoSlot) continue;
      const float now = fmaxf(top, s), old = expf(top - now), w = expf(s - now);
      top = now;
      sum = sum * old + w;
#pragma unroll
      for (int i = 0; i < L; ++i) acc[i] = acc[i] * old + w * to_float(static_cast<const T*>(a.v_pages)[int64_t(at) * 8 + i * 32 + lane]);
    }
    if (lane == 0) { max_s[warp] = top; sum_s[warp] = sum; }
#pragma unroll
    for (int i = 0; i < L; ++i) acc_s[warp][i * 32 + lane] = acc[i];
    __syncthreads();
    float all = -INFINITY, total = 0.f;
    for (int w = 0; w < kSimpleWarps; ++w) all = fmaxf(all, max_s[w]);
    for (int w = 0; w < kSimpleWarps; ++w) total += max_s[w] > -INFINITY ? sum_s[w] * expf(max_s[w] - all) : 0.f;
    for (int i = threadIdx.x; i < D; i += blockDim.x) {
      float value = 0.f;
      for (int w = 0; w < kSimpleWarps; ++w) value += max_s[w] > -INFINITY ? acc_s[w][i] * expf(max_s[w] - all) : 0.f;
      static_cast<T*>(a.out)[(int64_t(m) * a.q_heads + head) * D + i] = from_float<T>(length > 0 && total != 0.f ? value / total : 0.f);
    }
    if (threadIdx.x == 0) { norm_s[2 * g] = all; norm_s[2 * g + 1] = total; }
  }
  if (a.weights == nullptr) return;
  for (int g = 0; g < group; ++g) {
    load_query(kv * group + g);
    for (int p = warp; p < length; p += kSimpleWarps) {
      uint32_t at;
      const float s = score(p, at);
      if (at != kNoSlot && lane == 0) a.weights[a.layout.weight_of(table, a.kv_heads, kv, p)] += expf(s - norm_s[2 * g]) / norm_s[2 * g + 1];
    }
  }
}

template <typename T, int D>
int launch(const AttentionArguments& a, int M, void* stream) {
  const cudaError_t launched = launch_dependent(paged_attention_simple_kernel<T, D>, dim3(a.kv_heads, M), dim3(kSimpleWarps * 32),
                                                size_t(a.q_heads / a.kv_heads) * 8, stream, a);
  if (launched != cudaSuccess) return cuda_fail(launched, "paged attention launch");
  return MKB_OK;
}

int dispatch(const AttentionArguments& a, int M, int head_dim, int dtype, void* stream) {
  if (dtype == MKB_F16) {
    switch (head_dim) {
      case 64: return launch<__half, 64>(a, M, stream);
      case 128: return launch<__half, 128>(a, M, stream);
      case 192: return launch<__half, 192>(a, M, stream);
      default: return launch<__half, 256>(a, M, stream);
    }
  }
  switch (head_dim) {
    case 64: return launch<__nv_bfloat16, 64>(a, M, stream);
    case 128: return launch<__nv_bfloat16, 128>(a, M, stream);
    case 192: return launch<__nv_bfloat16, 192>(a, M, stream);
    default: return launch<__nv_bfloat16, 256>(a, M, stream);
  }
}

int check(const char* what, const void* q, const int* lengths, const void* out, const float* weights, int M, int q_heads,
          int kv_heads, int head_dim, int64_t q_row, int64_t q_head, int dtype, float scale, const void* workspace,
          int64_t workspace_bytes, int64_t need) {
  MKB_REQUIRE(q && lengths && out, MKB_E_ARGUMENT, "%s: null pointer", what);
  MKB_REQUIRE(q_heads > 0 && q_heads % kv_heads == 0, MKB_E_ARGUMENT, "%s: %d query heads for %d key-value heads", what, q_heads, kv_heads);
  MKB_REQUIRE(dtype == MKB_F16 || dtype == MKB_BF16, MKB_E_UNSUPPORTED, "%s: dtype tag %d (fp16 and bf16 supported)", what, dtype);
  MKB_REQUIRE(M <= 65535 && kv_heads <= 65535 && q_heads <= 1 << 20, MKB_E_UNSUPPORTED, "%s: %d sequences of %d heads", what, M, q_heads);
  MKB_REQUIRE(scale == scale && fabsf(scale) < INFINITY, MKB_E_ARGUMENT, "%s: scale is not finite", what);
  MKB_REQUIRE(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15) == 0 && q_row % 8 == 0 && q_head % 8 == 0,
              MKB_E_ALIGNMENT, "%s: queries and outputs lie on 16-byte vectors", what);
  MKB_REQUIRE(workspace_bytes >= need && (need == 0 || (workspace != nullptr && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0)),
              MKB_E_ARGUMENT, "%s: workspace of %lld bytes, %lld needed", what, (long long)workspace_bytes, (long long)need);
  return MKB_OK;
}

}  // namespace

int paged_layout(PagedLayout* layout, const char* what, const void* k_pages, const void* v_pages, const int* tables, int kv_heads,
                 int head_dim, int page, int columns, int64_t pages, int64_t page_stride, int64_t head_stride,
                 int64_t slot_stride, int64_t table_stride) {
  MKB_REQUIRE(kv_heads > 0 && page > 0 && columns > 0 && pages > 0 && pages < (int64_t(1) << 31) && table_stride >= 0, MKB_E_ARGUMENT,
              "%s: bad shape", what);
  MKB_REQUIRE(k_pages && v_pages && tables, MKB_E_ARGUMENT, "%s: null pointer", what);
  MKB_REQUIRE(head_dim > 0 && head_dim % 64 == 0 && head_dim <= 256, MKB_E_UNSUPPORTED, "%s: head_dim %d (64, 128, 192 and 256 supported)",
              what, head_dim);
  MKB_REQUIRE(int64_t(columns) * page < (int64_t(1) << 30), MKB_E_UNSUPPORTED, "%s: %d pages of %d slots per sequence", what, columns, page);
  MKB_REQUIRE(page_stride >= 0 && head_stride >= 0 && slot_stride >= 0, MKB_E_ARGUMENT, "%s: negative stride", what);
  MKB_REQUIRE(((reinterpret_cast<uintptr_t>(k_pages) | reinterpret_cast<uintptr_t>(v_pages)) & 15) == 0 && page_stride % 8 == 0 &&
                  head_stride % 8 == 0 && slot_stride % 8 == 0,
              MKB_E_ALIGNMENT, "%s: pages lie on 16-byte vectors", what);
  const int64_t extent = (pages - 1) * page_stride / 8 + (kv_heads - 1) * head_stride / 8 + (page - 1) * slot_stride / 8 + head_dim / 8;
  MKB_REQUIRE(page_stride / 8 < (int64_t(1) << 32) && extent < (int64_t(1) << 32), MKB_E_UNSUPPORTED, "%s: a pool spans 64 GiB or more", what);
  *layout = {tables, table_stride, FastDivide::of(uint32_t(page)), uint32_t(pages), uint32_t(columns), uint32_t(page_stride / 8),
             uint32_t(head_stride / 8), uint32_t(slot_stride / 8)};
  return MKB_OK;
}

cudaError_t take_paged_attention_status(unsigned int* value) {
  const unsigned int zero = 0;
  cudaError_t done = cudaMemcpyFromSymbol(value, g_paged_attention_status, sizeof(*value));
  if (done == cudaSuccess && *value != 0) done = cudaMemcpyToSymbol(g_paged_attention_status, &zero, sizeof(zero));
  return done;
}

}  // namespace mkb

extern "C" int64_t mkb_paged_attention_workspace_bytes(int M, int q_heads, int kv_heads, int head_dim, int page, int columns,
                                                       int with_weights) {
  if (M <= 0 || q_heads <= 0 || kv_heads <= 0 || head_dim <= 0 || page <= 0 || columns <= 0) return 0;
  return 0;
}

extern "C" int mkb_paged_attention_decode(const void* q, const int* lengths, const void* k_pages, const void* v_pages,
                                          const int* tables, void* out, float* weights, int M, int q_heads, int kv_heads,
                                          int head_dim, int page, int columns, int64_t pages, int64_t page_stride,
                                          int64_t head_stride, int64_t slot_stride, int64_t table_stride, int64_t q_row_stride,
                                          int64_t q_head_stride, float scale, int dtype, void* workspace, int64_t workspace_bytes,
                                          void* stream) {
  using namespace mkb;
  const char* what = "paged_attention_decode";
  MKB_REQUIRE(M >= 0, MKB_E_ARGUMENT, "%s: bad shape", what);
  if (M == 0) return MKB_OK;
  AttentionArguments a{};
  int status = paged_layout(&a.layout, what, k_pages, v_pages, tables, kv_heads, head_dim, page, columns, pages, page_stride, head_stride,
                            slot_stride, table_stride);
  if (status != MKB_OK) return status;
  status = check(what, q, lengths, out, weights, M, q_heads, kv_heads, head_dim, q_row_stride, q_head_stride, dtype, scale, workspace,
                 workspace_bytes, mkb_paged_attention_workspace_bytes(M, q_heads, kv_heads, head_dim, page, columns, weights != nullptr));
  if (status != MKB_OK) return status;
  a.q = q; a.lengths = lengths; a.k_pages = const_cast<void*>(k_pages); a.v_pages = const_cast<void*>(v_pages); a.out = out;
  a.weights = weights; a.q_row = q_row_stride; a.q_head = q_head_stride; a.q_heads = q_heads; a.kv_heads = kv_heads; a.scale = scale;
  return dispatch(a, M, head_dim, dtype, stream);
}

extern "C" int mkb_paged_rope_attention_decode(const void* qkv, const int* positions, const int* lengths, void* k_pages, void* v_pages,
                                               const int* tables, void* out, float* weights, int M, int q_heads, int kv_heads,
                                               int head_dim, int page, int columns, int64_t pages, int64_t page_stride,
                                               int64_t head_stride, int64_t slot_stride, int64_t table_stride, int64_t qkv_row_stride,
                                               float theta, float scale, int dtype, void* workspace, int64_t workspace_bytes,
                                               void* stream) {
  using namespace mkb;
  const char* what = "paged_rope_attention_decode";
  MKB_REQUIRE(M >= 0, MKB_E_ARGUMENT, "%s: bad shape", what);
  if (M == 0) return MKB_OK;
  AttentionArguments a{};
  int status = paged_layout(&a.layout, what, k_pages, v_pages, tables, kv_heads, head_dim, page, columns, pages, page_stride, head_stride,
                            slot_stride, table_stride);
  if (status != MKB_OK) return status;
  MKB_REQUIRE(positions, MKB_E_ARGUMENT, "%s: null pointer", what);
  MKB_REQUIRE(theta > 0.f && theta < INFINITY, MKB_E_ARGUMENT, "%s: theta is not positive", what);
  status = check(what, qkv, lengths, out, weights, M, q_heads, kv_heads, head_dim, qkv_row_stride, head_dim, dtype, scale, workspace,
                 workspace_bytes, mkb_paged_attention_workspace_bytes(M, q_heads, kv_heads, head_dim, page, columns, weights != nullptr));
  if (status != MKB_OK) return status;
  a.q = qkv; a.positions = positions; a.lengths = lengths; a.k_pages = k_pages; a.v_pages = v_pages; a.out = out; a.weights = weights;
  a.q_row = qkv_row_stride; a.q_head = head_dim; a.q_heads = q_heads; a.kv_heads = kv_heads; a.rope = 1; a.theta = theta; a.scale = scale;
  return dispatch(a, M, head_dim, dtype, stream);
}
