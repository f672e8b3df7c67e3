// Eviction from a paged key-value cache by accumulated attention weight.  Of a sequence of n slots a head keeps
// min(n, budget): the first `sinks`, the last `recent`, and of the others the heaviest, a tie going to the lower slot.  The
// kept slots, in their order, move to fresh pages with their keys, values and weights, so a page that other sequences read
// as well stays as it is, and no move waits for another.
#include <atomic>

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
constexpr int kHeldKeys = 49152;      // keys of a sequence that lie in shared memory; longer ones are read again for each digit

// One CTA per (head, sequence).  The border between kept and dropped weights is found digit by digit, most significant
// first: a histogram of the candidates that share the digits found so far says in which bin the last kept weight lies.  A
// warp's equal digits are counted by one of its lanes: many slots have the same small weight, or one of a few exponents, and
// queued at their bin.  Then every warp lists what it keeps of its own run of slots.  What bounds it is the chain of four
// digits for a CTA of 16 keys a thread, 25 of the 110 us for 16 x 8 sequences of up to 16384 slots; digits of 12 and 10 bits
// with the counts queueing, or with only the most common digit of a warp counted by a vote, measured no better, and a
// cluster of two CTAs with half of the slots each 116.
__global__ void __launch_bounds__(kSelectThreads) evict_select_kernel(PagedLayout layout, const float* __restrict__ weights,
                                                                      const int* __restrict__ lengths, int* __restrict__ kept,
                                                                      int kv_heads, int budget, int sinks, int recent, int held) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  extern __shared__ uint32_t key_s[];      // [held]
  __shared__ uint32_t bins_s[256];
  __shared__ uint32_t count_s[kSelectWarps][2];
  __shared__ uint32_t found_s[3];
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
  auto read_key = [&](int p) {
    const int64_t at = layout.weight_of(table, kv_heads, head, p);
    if (at < 0) {
      atomicOr(&g_paged_evict_status, 1u);
      return 0u;
    }
    return key_of(__ldg(weights + at));
  };
  const bool all_held = high <= held;
  if (all_held) {
    // eight at a time without a branch between them, so that their page numbers, then their weights, are under way together
    constexpr int kDeep = 8;
    bool missing = false;
    for (int p = low + int(threadIdx.x); p < high; p += kDeep * kSelectThreads) {
      int64_t at[kDeep];
      float read[kDeep];
#pragma unroll
      for (int u = 0; u < kDeep; ++u) at[u] = layout.weight_of(table, kv_heads, head, min(p + u * kSelectThreads, high - 1));
#pragma unroll
      for (int u = 0; u < kDeep; ++u) read[u] = __ldg(weights + max(at[u], int64_t(0)));
#pragma unroll
      for (int u = 0; u < kDeep; ++u) {
        missing |= at[u] < 0;
        if (p + u * kSelectThreads < high) key_s[p + u * kSelectThreads] = at[u] < 0 ? 0u : key_of(read[u]);
      }
    }
    if (missing) atomicOr(&g_paged_evict_status, 1u);
  }
  auto key_at = [&](int p) { return all_held ? key_s[p] : read_key(p); };
  // keys over `edge` stay, and of those that equal it the first `want`
  uint32_t edge = 0xffffffffu;
  if (want == 0) {
    __syncthreads();
  } else {
    uint32_t prefix = 0;
#pragma unroll 1
    for (int shift = 24;; shift -= 8) {
      if (threadIdx.x < 256) bins_s[threadIdx.x] = 0;
      __syncthreads();
      for (int p = low + threadIdx.x; p - lane < high; p += kSelectThreads) {
        const uint32_t key = p < high ? key_at(p) : 0u;
        const bool counts = p < high && (shift == 24 || (key >> (shift + 8)) == prefix);
        const uint32_t digit = counts ? (key >> shift) & 255u : 256u;
        const uint32_t same = __match_any_sync(0xffffffffu, digit);
        if (counts && lane == __ffs(same) - 1) atomicAdd(&bins_s[digit], __popc(same));
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
          if (before < uint32_t(want) && before + bin[i] >= uint32_t(want)) { found_s[0] = 255 - 8 * lane - i; found_s[1] = before; found_s[2] = bin[i]; }
          before += bin[i];
        }
      }
      __syncthreads();
      prefix = prefix << 8 | found_s[0];
      want -= int(found_s[1]);
      const bool whole_bin = found_s[2] == uint32_t(want);
      if (shift == 0) {
        edge = prefix;
        break;
      }
      if (whole_bin) {      // everything with these digits stays: no key is lower than the one before them
        edge = (prefix << shift) - 1;
        want = 0;
        break;
      }
      __syncthreads();
    }
  }
  const int run = (n + kSelectThreads - 1) / kSelectThreads * 32;
  const int first = warp * run, last = min(first + run, n);
  const bool chosen = budget > sinks + recent;
  auto sort_out = [&](int p, bool& over, bool& level) {
    over = level = false;
    if (p >= last) return;
    if (p < low || p >= high) { over = true; return; }
    const uint32_t key = key_at(p);
    over = chosen && key > edge;
    level = key == edge;
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
constexpr int kMoveRows = 64;     // of a block
constexpr int kMoveDeep = 4;      // vectors of keys, and of values, of a thread under way

// A block looks up where its rows come from and go to, a thread for each, moving their weights; then its threads move the
// rows' 16-byte vectors.  (The look-up by each thread for its own vectors made every copy wait for three loads in turn: 110
// us for 16 x 8 x 4096 rows of 256 bytes, against 78 at the copy rate.)  Bound by memory: 4 * head_dim bytes read and as many written
// for a row, which are not read again soon, so they pass the caches as streams.
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(PagedLayout from, PagedLayout to, uint4* __restrict__ k_pages,
                                                                  uint4* __restrict__ v_pages, float* __restrict__ weights,
                                                                  const int* __restrict__ kept, int kv_heads, int budget, int vectors) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  __shared__ uint2 move_s[kMoveRows];     // source and target, in vectors
  const int head = blockIdx.y, m = blockIdx.z, row0 = blockIdx.x * kMoveRows;
  const int rows = min(kMoveRows, budget - row0);
  if (int(threadIdx.x) < rows) {
    const int row = row0 + threadIdx.x, old = __ldg(kept + (int64_t(m) * kv_heads + head) * budget + row);
    uint2 move = make_uint2(kNoSlot, kNoSlot);
    if (old >= 0) {
      const int* old_table = from.tables + m * from.table_stride;
      const int* new_table = to.tables + m * to.table_stride;
      move = make_uint2(from.vector_of(old_table, head, old), to.vector_of(new_table, head, row));
      if (move.x == kNoSlot || move.y == kNoSlot) {
        atomicOr(&g_paged_evict_status, 1u);
        move.x = kNoSlot;
      } else {
        weights[to.weight_of(new_table, kv_heads, head, row)] = weights[from.weight_of(old_table, kv_heads, head, old)];
      }
    }
    move_s[threadIdx.x] = move;
  }
  __syncthreads();
  const int total = rows * vectors;
  for (int start = threadIdx.x; start < total; start += kMoveDeep * kMoveThreads) {
    uint4 key[kMoveDeep], value[kMoveDeep];
    int64_t target[kMoveDeep];
#pragma unroll
    for (int i = 0; i < kMoveDeep; ++i) {
      const int index = start + i * kMoveThreads, row = index / vectors;
      target[i] = -1;
      if (index >= total) continue;
      const uint2 move = move_s[row];
      if (move.x == kNoSlot) continue;
      const int vector = index - row * vectors;
      key[i] = __ldcs(k_pages + (int64_t(move.x) + vector));
      value[i] = __ldcs(v_pages + (int64_t(move.x) + vector));
      target[i] = int64_t(move.y) + vector;
    }
#pragma unroll
    for (int i = 0; i < kMoveDeep; ++i)
      if (target[i] >= 0) {
        __stcs(k_pages + target[i], key[i]);
        __stcs(v_pages + target[i], value[i]);
      }
  }
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
  const int64_t capacity = int64_t(columns) * page;
  const int held = capacity < kHeldKeys ? int(capacity) : kHeldKeys;
  int device = 0;
  cudaGetDevice(&device);
  static std::atomic<uint64_t> opted{0};
  if (!(opted.load(std::memory_order_acquire) >> (device & 63) & 1)) {
    const cudaError_t set = cudaFuncSetAttribute(evict_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kHeldKeys * 4);
    if (set != cudaSuccess) return cuda_fail(set, "paged evict shared memory");
    opted.fetch_or(uint64_t(1) << (device & 63), std::memory_order_release);
  }
  cudaError_t launched = launch_dependent(evict_select_kernel, dim3(kv_heads, M), dim3(kSelectThreads), size_t(held) * 4, stream, from,
                                          static_cast<const float*>(weights), lengths, kept, kv_heads, budget, sinks, recent, held);
  if (launched != cudaSuccess) return cuda_fail(launched, "paged evict launch");
  launched = launch_dependent(evict_move_kernel, dim3(unsigned((int64_t(budget) + kMoveRows - 1) / kMoveRows), kv_heads, M), dim3(kMoveThreads), 0, stream,
                              from, to, static_cast<uint4*>(k_pages), static_cast<uint4*>(v_pages), weights,
                              static_cast<const int*>(kept), kv_heads, budget, head_dim / 8);
  if (launched != cudaSuccess) return cuda_fail(launched, "paged evict launch");
  return MKB_OK;
}
