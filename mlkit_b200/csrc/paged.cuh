// What the operators over a paged key-value cache share: the layout, the way from a slot to its address, the status word.
//
// A cache is a pool of pages [pages, kv_heads, page, head_dim] (any strides of whole 16-byte vectors, keys and values
// alike) and a table of page numbers per sequence: slot p of a sequence lies at slot p % page of page table[p / page].
#pragma once

#include "mkb_common.cuh"

namespace mkb {

// n / d for n < 2^31 by a multiplication (round-up method of Granlund and Montgomery, 1994).
struct FastDivide {
  uint32_t divisor, multiplier, shift;
  static FastDivide of(uint32_t d) {
    uint32_t shift = 0;
    while ((uint64_t(1) << shift) < d) ++shift;
    return {d, uint32_t(((uint64_t(1) << 32) * ((uint64_t(1) << shift) - d)) / d + 1), shift};
  }
  __device__ __forceinline__ uint32_t quotient(uint32_t n) const { return (__umulhi(n, multiplier) + n) >> shift; }
};

constexpr uint32_t kNoSlot = 0xffffffffu;

struct PagedLayout {
  const int* tables;
  int64_t table_stride;
  FastDivide page;
  uint32_t pages, columns;
  uint32_t page_stride, head_stride, slot_stride;   // in 16-byte vectors: a pool of up to 2^32 - 1 of them has 32-bit offsets

  // Offset of (sequence, head, slot) in 16-byte vectors; kNoSlot when the table names no page of the pool.
  __device__ __forceinline__ uint32_t vector_of(const int* table, uint32_t head, uint32_t slot) const {
    const uint32_t column = page.quotient(slot);
    const uint32_t id = uint32_t(__ldg(table + column));
    return id < pages ? id * page_stride + head * head_stride + (slot - column * page.divisor) * slot_stride : kNoSlot;
  }
  // Number of (sequence, head, slot) in an accumulator [pages, heads, page]; -1 as above.  Early: before the wait for the
  // kernel before, when the first-level cache may still hold what an earlier kernel read.
  template <bool Early = false>
  __device__ __forceinline__ int64_t weight_of(const int* table, uint32_t heads, uint32_t head, uint32_t slot) const {
    const uint32_t column = page.quotient(slot);
    const uint32_t id = uint32_t(Early ? __ldcg(table + column) : __ldg(table + column));
    return id < pages ? (int64_t(id) * heads + head) * page.divisor + (slot - column * page.divisor) : -1;
  }
  __device__ __forceinline__ int capacity() const { return int(columns * page.divisor); }
};

// Fills `layout` after checking it; `what` names the caller in the error text.
int paged_layout(PagedLayout* layout, const char* what, const void* k_pages, const void* v_pages, const int* tables, int kv_heads,
                 int head_dim, int page, int columns, int64_t pages, int64_t page_stride, int64_t head_stride,
                 int64_t slot_stride, int64_t table_stride);

// Read and clear the status words of the operators' files.
cudaError_t take_paged_attention_status(unsigned int* value);
cudaError_t take_paged_evict_status(unsigned int* value);

}  // namespace mkb
