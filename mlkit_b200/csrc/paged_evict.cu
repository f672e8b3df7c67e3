// Eviction from a paged key-value cache by accumulated attention weight.  Of a sequence of n slots a head keeps
// min(n, budget): the first `sinks`, the last `recent`, and of the others the heaviest, a tie going to the lower slot.  The
// kept slots, in their order, move to fresh pages with their keys, values and weights, so a page that other sequences read
// as well stays as it is, and no move waits for another.
#include "paged.cuh"

namespace mkb {
namespace {

__device__ unsigned int g_paged_evict_status = 0;

// A monotone map of a weight to an unsigned word: negative zero equals zero, a NaN ranks below everything.
__device__ __forceinline__ uint32_t key_of(float weight) {
  const uint32_t bits = __float_as_uint(weight);
  if ((bits & 0x7fffffffu) > 0x7f800000u) return 0u;
  if ((bits & 0x7fffffffu) == 0u) return 0x80000000u;
  return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

constexpr int kSelectThreads = 1024;
constexpr int kSelectWarps = kSelectThreads / 32;

// One CTA per (head, sequence).  The border between kept and dropped weights is found digit by digit, most significant
// first: a histogram of the candidates that share the digits found so far says in which bin the last kept weight lies.
// Then every warp lists what it keeps of its own run of slots.
__global__ void __launch_bounds__(kSelectThreads) evict_select_kernel(PagedLayout layout, const float* __restrict__ weights,
                                                                      const int* __restrict__ lengths, int* __restrict__ kept,
                                                                      int kv_heads, int budget, int sinks, int recent) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  __shared__ uint32_t bins_s[256];
  __shared__ uint32_t count_s[kSelectWarps][2];
  __shared__ uint32_t found_s[2];
  const int head = blockIdx.x, m = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int* table = layout.tables + m * layout.table_stride;
  int* list = kept + (int64_t(m) * kv_heads + head) * budget;
  int n = lengths[m];
  if (n > layout.capacity()) {
    if (threadIdx.x == 0) atomicOr(&g_paged_evict_status, 1u);
    n = layout.capacity();
  }
  n = max(n, 0);
  if (n <= budget) {
    for (int j = threadIdx.x; j < budget; j += kSelectThreads) list[j] = j < n ? j : -1;
    return;
  }
  const int low = sinks, high = n - recent;          // candidates: [low, high)
  int want = budget - sinks - recent;                // of which this many stay
  auto key_at = [&](int p) {
    const int64_t at = layout.weight_of(table, kv_heads, head, p);
    if (at < 0) {
      atomicOr(&g_paged_evict_status, 1u);
      return 0u;
    }
    return key_of(weights[at]);
  };
  uint32_t prefix = 0;
#pragma unroll 1
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < 256; i += kSelectThreads) bins_s[i] = 0;
    __syncthreads();
    for (int p = low + threadIdx.x; p < high; p += kSelectThreads) {
      const uint32_t key = key_at(p);
      if (shift == 24 || (key >> (shift + 8)) == prefix) atomicAdd(&bins_s[(key >> shift) & 255u], 1u);
    }
    __syncthreads();
    if (warp == 0) {   // lane l holds bins 255 - 8l down to 248 - 8l: a scan from the heaviest bin
      uint32_t own = 0, bin[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) own += bin[i] = bins_s[255 - 8 * lane - i];
      uint32_t before = own;
#pragma unroll
      for (int step = 1; step < 32; step <<= 1) {
        const uint32_t other = __shfl_up_sync(0xffffffffu, before, step);
        if (lane >= step) before += other;
      }
      before -= own;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (before < uint32_t(want) && before + bin[i] >= uint32_t(want)) { found_s[0] = 255 - 8 * lane - i; found_s[1] = before; }
        before += bin[i];
      }
      if (want == 0 && lane == 0) { found_s[0] = 255; found_s[1] = 0; }
    }
    __syncthreads();
    prefix = prefix << 8 | found_s[0];
    want -= int(found_s[1]);
    __syncthreads();
  }
  // prefix: the lightest weight kept; `want`: how many of those that equal it stay (none when nothing but the safe slots does)
  const int run = (n + kSelectThreads - 1) / kSelectThreads * 32;
  const int first = warp * run, last = min(first + run, n);
  auto sort_out = [&](int p, bool& over, bool& level) {
    over = level = false;
    if (p >= last) return;
    if (p < low || p >= high) { over = true; return; }
    const uint32_t key = key_at(p);
    over = key > prefix && budget > sinks + recent;
    level = key == prefix;
  };
  uint32_t overs = 0, levels = 0;
  bool over, level;
  for (int p = first; p < last; p += 32) {
    sort_out(p + lane, over, level);
    overs += __popc(__ballot_sync(0xffffffffu, over));
    levels += __popc(__ballot_sync(0xffffffffu, level));
  }
  if (lane == 0) { count_s[warp][0] = overs; count_s[warp][1] = levels; }
  __syncthreads();
  overs = levels = 0;
  for (int w = 0; w < warp; ++w) { overs += count_s[w][0]; levels += count_s[w][1]; }
  const uint32_t below = (1u << lane) - 1;
  for (int p = first; p < last; p += 32) {
    sort_out(p + lane, over, level);
    const uint32_t over_mask = __ballot_sync(0xffffffffu, over), level_mask = __ballot_sync(0xffffffffu, level);
    const uint32_t over_rank = overs + __popc(over_mask & below), level_rank = levels + __popc(level_mask & below);
    if (over || (level && level_rank < uint32_t(want))) list[over_rank + min(level_rank, uint32_t(want))] = p + lane;
    overs += __popc(over_mask);
    levels += __popc(level_mask);
  }
}

constexpr int kMoveThreads = 256;

// A thread moves one 16-byte vector of a key and of a value.
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(PagedLayout from, PagedLayout to, uint4* __restrict__ k_pages,
                                                                  uint4* __restrict__ v_pages, float* __restrict__ weights,
                                                                  const int* __restrict__ kept, int kv_heads, int budget, int vectors) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int head = blockIdx.y, m = blockIdx.z;
  const uint32_t index = blockIdx.x * kMoveThreads + threadIdx.x;
  const uint32_t row = index / vectors, vector = index - row * vectors;
  if (row >= uint32_t(budget)) return;
  const int old = kept[(int64_t(m) * kv_heads + head) * budget + row];
  if (old < 0) return;
  const int* old_table = from.tables + m * from.table_stride;
  const int* new_table = to.tables + m * to.table_stride;
  const uint32_t source = from.vector_of(old_table, head, old), target = to.vector_of(new_table, head, row);
  if (source == kNoSlot || target == kNoSlot) {
    atomicOr(&g_paged_evict_status, 1u);
    return;
  }
  k_pages[int64_t(target) + vector] = k_pages[int64_t(source) + vector];
  v_pages[int64_t(target) + vector] = v_pages[int64_t(source) + vector];
  if (vector == 0) weights[to.weight_of(new_table, kv_heads, head, row)] = weights[from.weight_of(old_table, kv_heads, head, old)];
}

}  // namespace

cudaError_t take_paged_evict_status(unsigned int* value) {
  const unsigned int zero = 0;
  cudaError_t done = cudaMemcpyFromSymbol(value, g_paged_evict_status, sizeof(*value));
  if (done == cudaSuccess && *value != 0) done = cudaMemcpyToSymbol(g_paged_evict_status, &zero, sizeof(zero));
  return done;
}

}  // namespace mkb

extern "C" int mkb_paged_evict(void* k_pages, void* v_pages, float* weights, const int* tables, const int* lengths,
                               const int* new_tables, int* kept, int M, int kv_heads, int head_dim, int page, int columns,
                               int new_columns, int64_t pages, int64_t page_stride, int64_t head_stride, int64_t slot_stride,
                               int64_t table_stride, int64_t new_table_stride, int budget, int sinks, int recent, void* stream) {
  using namespace mkb;
  const char* what = "paged_evict";
  MKB_REQUIRE(M >= 0 && budget > 0 && sinks >= 0 && recent >= 0, MKB_E_ARGUMENT, "%s: bad shape", what);
  MKB_REQUIRE(int64_t(sinks) + recent <= budget, MKB_E_ARGUMENT, "%s: %d first and %d last slots exceed the budget of %d", what, sinks, recent, budget);
  if (M == 0) return MKB_OK;
  MKB_REQUIRE(weights && lengths && kept, MKB_E_ARGUMENT, "%s: null pointer", what);
  MKB_REQUIRE(M <= 65535 && kv_heads <= 65535, MKB_E_UNSUPPORTED, "%s: %d sequences of %d heads", what, M, kv_heads);
  PagedLayout from, to;
  int status = paged_layout(&from, what, k_pages, v_pages, tables, kv_heads, head_dim, page, columns, pages, page_stride, head_stride,
                            slot_stride, table_stride);
  if (status != MKB_OK) return status;
  status = paged_layout(&to, what, k_pages, v_pages, new_tables, kv_heads, head_dim, page, new_columns, pages, page_stride, head_stride,
                        slot_stride, new_table_stride);
  if (status != MKB_OK) return status;
  MKB_REQUIRE(int64_t(new_columns) * page >= budget || int64_t(new_columns) * page >= int64_t(columns) * page, MKB_E_ARGUMENT,
              "%s: %d new pages of %d slots do not hold the budget of %d", what, new_columns, page, budget);
  cudaError_t launched = launch_dependent(evict_select_kernel, dim3(kv_heads, M), dim3(kSelectThreads), 0, stream, from,
                                          static_cast<const float*>(weights), lengths, kept, kv_heads, budget, sinks, recent);
  if (launched != cudaSuccess) return cuda_fail(launched, "paged evict launch");
  const int vectors = head_dim / 8;
  const int64_t blocks = (int64_t(budget) * vectors + kMoveThreads - 1) / kMoveThreads;
  launched = launch_dependent(evict_move_kernel, dim3(unsigned(blocks), kv_heads, M), dim3(kMoveThreads), 0, stream, from, to,
                              static_cast<uint4*>(k_pages), static_cast<uint4*>(v_pages), weights, static_cast<const int*>(kept),
                              kv_heads, budget, vectors);
  if (launched != cudaSuccess) return cuda_fail(launched, "paged evict launch");
  return MKB_OK;
}
