// Attention of one new token per sequence over a paged key-value cache.
//   s[h, p] = scale * q[h] . k[p],   w[h, p] = exp(s[h, p] - max) / sum,   out[h] = sum_p w[h, p] v[p]
// with the query heads h of a group sharing one key-value head; optionally acc[p] += sum over the group of w[h, p].
//
// What bounds it: reading the cache once, 4 * head_dim bytes a slot and key-value head for 4 * head_dim * group flops.  So:
// * Work is cut into tiles of 16 slots of one (sequence, key-value head); the tiles of all sequences in a row are dealt out
//   in equal runs to as many CTAs as the GPU holds, whatever the lengths.  A (sequence, head) that crosses from one CTA to
//   the next leaves partial (max, sum, output) triples in two slots per CTA.  Partials are joined in groups of eight CTAs,
//   then the groups: a ticket counts the arrivals and the CTA that comes last joins, always in the order of the CTAs, so
//   results do not depend on who that was, and leaves the ticket at zero.  (A second launch for the join measured as much on
//   the device, 3 to 6 us, and 3 us more on the host; one level of a hundred partials 13 us.)
// * A warp copies its own tiles into a ring of its own with cp.async, several tiles ahead, across the borders of
//   sequences, and waits for nobody else's.  A copy instruction takes whole rows (rows cut to the 64 bytes that a lane quad
//   feeds to the tensor core, which would spare the warp its barriers, measured 4.5 TB/s where whole ones measure 5.7, both
//   over the whole call).
//   Pieces of 16 bytes are swapped within 128 bytes by the row so that neither the reads of the keys, pieces t of rows g
//   (g = lane / 4, t = lane % 4), nor those of the values, pieces g of rows 2t, meet in a bank.  Which dimension stands at
//   which place of a product's reduction or of its rows is free as long as queries and outputs agree, so a lane feeds the
//   8 dimensions of a piece to two products and needs no ldmatrix.
// * Slots are the 16 rows of the tensor core's tile and the group's query heads its 8 columns: S^T = K Q^T, O^T = V^T P^T, so
//   eight heads leave nothing unused and the running maximum of a column is three shuffles.  P^T turns from the accumulator's
//   layout to the operand's with movmatrix.  More than eight heads of a group are several tiles of heads, which read the
//   cache again (from L2, mostly).
// * Rounding: products of 16-bit values are exact, all sums are fp32.  A softmax weight is held in two 16-bit parts (its
//   rounding and the rest) for the product with the values, scaled by 2^14 so that weights down to 2^-38 of the largest stay
//   within fp16's range: 2^-22 of it is left out in fp16 and 2^-17 in bf16, far below the step the output is rounded to.  So is a
//   rotated query: 2^-23 of a value (2^-24 absolute for small ones) in fp16, 2^-17 in bf16, of which a score is off by as much of
//   sum |q k|.  Weights that are accumulated are taken from the scores in fp32; for them a bf16 query has a third part, which
//   leaves out less than fp32 does.
// Measured (device time, launch included): 131071 slots of 8 key-value heads of 128, 64 query heads: 94 us, 5.7 TB/s of the
// measured 6.55; 64 sequences of 500 to 16384 slots, 32 query heads: 200 us, 6.0 TB/s; 8 sequences of 1024: 14 us.
#include <atomic>

#include "paged.cuh"

namespace mkb {
namespace {

__device__ unsigned int g_paged_attention_status = 0;

constexpr int kTile = 16;       // slots of a tile
constexpr int kHeads = 8;       // query heads of a tile
constexpr float kShift = 14.f;  // weights are held times 2^14

struct AttentionArguments {
  PagedLayout layout;
  const void* q;
  const int* positions;     // with a rotation
  const int* lengths;
  uint4* k_pages;
  uint4* v_pages;
  void* out;
  float* weights;
  int64_t q_row, q_head;    // strides in elements
  int rows, q_heads, kv_heads, group, head_tiles, ctas;
  FastDivide by_head_tiles;
  float theta, scale_log2;
  // workspace
  float* partial;           // [ctas][2][kHeads][head_dim]: of the item a CTA's run begins within, and of the one it ends within
  float2* partial_norm;     // [ctas][2][kHeads]: maximum (in powers of two), sum
  unsigned int* tickets;    // [ctas][3]: of the groups that begin with a CTA's two partials, of the item that crosses its end
  float* norm;              // [rows][q_heads]: log2 of the softmax's sum, with weights
  float* scores;            // [tiles][min(group, 8)][kTile], with weights
};

__device__ __forceinline__ uint32_t shared_address(const void* p) { return uint32_t(__cvta_generic_to_shared(p)); }

template <typename T> struct Types;
template <> struct Types<__half> {
  static constexpr float kRotated = 0.5f;   // of a rotated query is held: the turn of two values of 65504 is 92637 long
  static __device__ __forceinline__ float2 widen(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
  static __device__ __forceinline__ uint32_t narrow(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  static __device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};
template <> struct Types<__nv_bfloat16> {
  static constexpr float kRotated = 1.f;
  static __device__ __forceinline__ float2 widen(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  }
  static __device__ __forceinline__ uint32_t narrow(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  static __device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};

// 2^x; below 2^-126 it is 0.  The weights of a softmax and what fades them need no more.
__device__ __forceinline__ float power_of_two(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Two floats as a pair of 16-bit values and a pair of what their rounding left out.
template <typename T>
__device__ __forceinline__ void split(float lo, float hi, uint32_t& pair, uint32_t& rest) {
  pair = Types<T>::narrow(lo, hi);
  const float2 held = Types<T>::widen(pair);
  rest = Types<T>::narrow(lo - held.x, hi - held.y);
}

__device__ __forceinline__ uint32_t turn_matrix(uint32_t v) {   // an 8 x 8 matrix of 16-bit values across a warp, transposed
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// What of a sequence lies in the cache, and how many tiles it has with the token that this call adds.
struct Extent {
  int held, tiles, added;
};
template <bool Rope, bool Early = false>      // Early: as in PagedLayout
__device__ __forceinline__ Extent extent_of(const AttentionArguments& a, int m, bool& beyond) {
  const int n = Early ? __ldcg(a.lengths + m) : __ldg(a.lengths + m), capacity = a.layout.capacity();
  if (n < 0) return {0, 0, 0};
  const int added = Rope && n < capacity;
  if (n > capacity - Rope) beyond = true;
  const int held = min(n, capacity);
  return {held, (held + added + kTile - 1) / kTile, added};
}

// The tiles of all sequences, (sequence, head tile, tile) in order, dealt out in runs that differ by one at most; fewer than
// 2^31 of them.  `per_row`: head tiles of a sequence; `least`: tiles that a CTA should have.
struct Run {
  int begin, end, total;
  int each, more;                  // tiles of a CTA, and of how many CTAs have one more
  int row, head, tile;             // where the run begins
  // the CTA whose run holds a tile
  __device__ __forceinline__ int holder(int index) const {
    const int longer = more * (each + 1);
    return index < longer ? index / (each + 1) : more + (index - longer) / each;
  }
};
template <bool Rope, int Threads, bool Early = false>
__device__ __forceinline__ Run find_run(const AttentionArguments& a, int per_row, int least, int cta, int ctas) {
  __shared__ int warp_s[Threads / 32];
  __shared__ int found_s[3];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int share = (a.rows + Threads - 1) / Threads;
  const int first = min(int(threadIdx.x) * share, a.rows), last = min(first + share, a.rows);
  bool beyond = false;
  int own = 0;
  for (int m = first; m < last; ++m) own += extent_of<Rope, Early>(a, m, beyond).tiles;
  if (beyond && cta == 0) atomicOr(&g_paged_attention_status, 1u);
  own *= per_row;
  int before = own;
#pragma unroll
  for (int step = 1; step < 32; step <<= 1) {
    const int other = __shfl_up_sync(0xffffffffu, before, step);
    if (lane >= step) before += other;
  }
  if (lane == 31) warp_s[warp] = before;
  __syncthreads();
  Run run;
  run.total = 0;
#pragma unroll
  for (int w = 0; w < Threads / 32; ++w) {
    if (w < warp) before += warp_s[w];
    run.total += warp_s[w];
  }
  before -= own;
  const int active = min(ctas, max(1, (run.total + least - 1) / least));
  run.each = run.total / active;
  run.more = run.total - run.each * active;
  run.begin = cta < active ? cta * run.each + min(cta, run.more) : run.total;
  run.end = cta < active ? run.begin + run.each + (cta < run.more) : run.total;
  if (run.begin < run.end && before <= run.begin && run.begin < before + own) {
    int rest = run.begin - before;
    for (int m = first; m < last; ++m) {
      const Extent extent = extent_of<Rope, Early>(a, m, beyond);
      if (rest < extent.tiles * per_row) {
        found_s[0] = m;
        found_s[1] = rest / extent.tiles;
        found_s[2] = rest - found_s[1] * extent.tiles;
        break;
      }
      rest -= extent.tiles * per_row;
    }
  }
  __syncthreads();
  run.row = found_s[0]; run.head = found_s[1]; run.tile = found_s[2];
  return run;
}

// A place in the order of the tiles.
template <bool Rope, bool Early = false>
struct Cursor {
  int row, head, tile;
  Extent extent;
  // The length is read again (from L1) instead of handed on by find_run: what the compiler then knows of an extent, or
  // how it schedules the loop for it, measured 15 % of the whole (200 against 233 us for the ragged batch of 64).
  __device__ __forceinline__ Cursor(const AttentionArguments& a, const Run& run) : row(run.row), head(run.head), tile(run.tile) {
    bool beyond;
    extent = extent_of<Rope, Early>(a, row, beyond);
  }
  // `steps` tiles on; the caller keeps it within the run.
  __device__ __forceinline__ void advance(const AttentionArguments& a, int per_row, int steps) {
    tile += steps;
    while (tile >= extent.tiles) {
      tile -= extent.tiles;
      if (++head == per_row) {
        head = 0;
        bool beyond;
        do extent = extent_of<Rope, Early>(a, ++row, beyond); while (extent.tiles == 0);
      }
    }
  }
};

// CTAs of four warps an SM.  (One CTA of eight warps for heads of 128 measured 107 us where two of four measure 91; for heads of
// 64 without a rotation four CTAs 17 and 29 us where two measure 22 and 34, but with one, whose registers then do not
// suffice, 43 where two with six tiles a warp measure 38; heads of 192 and 256 with more warps of two tiles each, or with two
// CTAs of two warps, 5 to 15 % more.)
constexpr int ctas_of(int head_dim, bool rope) { return head_dim == 64 ? (rope ? 2 : 4) : head_dim == 128 ? 2 : 1; }

template <int D, bool Rope, bool Weighted> struct Shape {
  static constexpr int kWarps = 4;
  static constexpr int kStages = D == 64 && Rope ? 6 : 3;
  static constexpr int kCtas = ctas_of(D, Rope);                 // per SM
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kPieces = D / 8;                          // of 16 bytes in a row
  static constexpr int kOps = kTile * kPieces / 32;              // that a lane copies of the keys, and of the values
  static constexpr int kHalf = kTile * D * 2;                    // bytes of a tile's keys
  static constexpr int kStageBytes = 2 * kHalf;
  static __device__ __forceinline__ int key_at(int row, int piece) { return (row * kPieces + (piece ^ (row & 1) << 2)) * 16; }
  static __device__ __forceinline__ int value_at(int row, int piece) { return kHalf + (row * kPieces + (piece ^ (row & 6))) * 16; }
  static constexpr int kRowFloats = D + 4;                       // of the outputs where the warps meet
  static constexpr int kRing = 0;
  static constexpr int kValid = kRing + kWarps * kStages * kStageBytes;     // [warp][stage]: which of a tile's slots count
  static constexpr int kNorm = kValid + kWarps * kStages * 4;               // [warp][head] float2
  static constexpr int kMeet = kNorm + kWarps * kHeads * 8;                 // [warp]: the stage that holds its outputs
  static constexpr int kTicket = kMeet + kWarps * 4;
  static constexpr int kTurns = (kTicket + 4 + 15) / 16 * 16;               // [D / 2] double: turns per position
  static constexpr int kCosine = kTurns + D / 2 * 8;                        // [D / 2][2] float
  static constexpr int kExact = kCosine + D / 2 * 8;                        // [D / 2][2] double
  static constexpr int kThird = kExact + D / 2 * 16;                        // [warp][D / 32][lane] uint4: third parts of rotated queries
  static constexpr int kBytes = kThird + (Weighted ? kWarps * D * 16 : 0);
  static_assert(kBytes + 1024 <= 233472 / kCtas, "shared memory");
  static_assert(kHeads * kRowFloats * 4 <= kStageBytes, "a warp's outputs fit a stage");
};

constexpr int kGroup = 8;      // partials joined at a time

// Joins `count` partials of an item, of the CTAs left + first, left + first + step, ... (the tail slot of CTA `left`, the head
// slots of the others): into the output, or into the slot of the first.  A thread takes two pieces of four dimensions at a
// time, so that sixteen loads are under way.
template <typename T, int D, int Threads>
__device__ __forceinline__ void join(const AttentionArguments& a, int left, int first, int step, int count, int heads, int64_t out_row, bool final,
                                     float2* norm_s) {
  constexpr int kPieces = D / 4;
  auto slot_of = [&](int i) { return (int64_t(left + first + i * step) * 2 + (first + i == 0)) * kHeads; };
#pragma unroll 1
  for (int index = threadIdx.x; index < heads * kPieces; index += 2 * Threads) {
    float top[2] = {-INFINITY, -INFINITY}, total[2] = {0.f, 0.f}, x[2][4] = {};
    int head[2], d[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int piece = min(index + u * Threads, heads * kPieces - 1);
      head[u] = piece / kPieces;
      d[u] = (piece - head[u] * kPieces) * 4;
    }
#pragma unroll 1
    for (int base = 0; base < count; base += kGroup) {
      float2 norm[kGroup][2];
      float4 v[kGroup][2];
#pragma unroll
      for (int i = 0; i < kGroup; ++i)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int64_t slot = slot_of(min(base + i, count - 1)) + head[u];
          norm[i][u] = __ldcg(a.partial_norm + slot);
          v[i][u] = __ldcg(reinterpret_cast<const float4*>(a.partial + slot * D + d[u]));
        }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float now = top[u];
#pragma unroll
        for (int i = 0; i < kGroup; ++i) now = fmaxf(now, norm[i][u].x);
        const float fade = total[u] == 0.f ? 0.f : power_of_two(top[u] - now);
        top[u] = now;
        total[u] *= fade;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[u][e] *= fade;
#pragma unroll
        for (int i = 0; i < kGroup; ++i) {
          if (base + i >= count || norm[i][u].y == 0.f) continue;
          const float share = power_of_two(norm[i][u].x - now);
          total[u] += norm[i][u].y * share;
          x[u][0] += v[i][u].x * share; x[u][1] += v[i][u].y * share; x[u][2] += v[i][u].z * share; x[u][3] += v[i][u].w * share;
        }
      }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (index + u * Threads >= heads * kPieces) continue;
      if (final) {
        const float inverse = total[u] == 0.f ? 0.f : 1.f / total[u];
        *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + (out_row + head[u]) * D + d[u]) =
            make_uint2(Types<T>::narrow(x[u][0] * inverse, x[u][1] * inverse), Types<T>::narrow(x[u][2] * inverse, x[u][3] * inverse));
        if (a.weights != nullptr && d[u] == 0) a.norm[out_row + head[u]] = top[u] - kShift + log2f(total[u]);
      } else {
        *reinterpret_cast<float4*>(a.partial + (slot_of(0) + head[u]) * D + d[u]) = make_float4(x[u][0], x[u][1], x[u][2], x[u][3]);
        if (d[u] == 0) norm_s[head[u]] = make_float2(top[u], total[u]);
      }
    }
  }
  if (!final) {    // the sums last: the other threads of a head have read them
    __syncthreads();
    if (int(threadIdx.x) < heads) a.partial_norm[slot_of(0) + threadIdx.x] = norm_s[threadIdx.x];
  }
}

// Whether this CTA is the last of `count` to come to a ticket, which is then zero again.  What the others wrote before is
// there for all threads.
__device__ __forceinline__ bool last_of(unsigned int* ticket, int count, unsigned int* shared) {
  __syncthreads();
  if (threadIdx.x == 0) {
    unsigned int before;
    asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(before) : "l"(ticket) : "memory");
    if (before == unsigned(count - 1)) *ticket = 0;
    *shared = before;
  }
  __syncthreads();
  return *shared == unsigned(count - 1);
}

// Weighted: weights are accumulated, for which rotated bf16 queries are held in a third part.  Of no use to the output, which is
// rounded to 2^-8, and not free: eight sequences of 1024, 32 query heads of 128: 14.7 us where two parts take 13.9, of 3000
// to 6000, heads of 192: 50 and 44, of 256: 61 and 55 (the ragged batch of 64 measured no difference).
template <typename T, int D, bool Rope, bool Weighted>
__global__ void __launch_bounds__(Shape<D, Rope, Weighted>::kThreads, Shape<D, Rope, Weighted>::kCtas) paged_attention_kernel(AttentionArguments a) {
  using S = Shape<D, Rope, Weighted>;
  using Y = Types<T>;
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, cta = blockIdx.x;
  const int per_row = a.kv_heads * a.head_tiles;
  double* turns_s = reinterpret_cast<double*>(smem + S::kTurns);
  float2* cosine_s = reinterpret_cast<float2*>(smem + S::kCosine);
  double2* exact_s = reinterpret_cast<double2*>(smem + S::kExact);
  if (Rope)   // the angle in 64 bits: a far position times a frequency rounded to 32 bits is off by hundredths of a turn
    for (int i = threadIdx.x; i < D / 2; i += S::kThreads)
      turns_s[i] = exp2(-log2(double(a.theta)) * double(i) / double(D / 2)) * 0.15915494309189533577;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // only now: what a dependent kernel reads before its own wait, the lengths and tables, is then there
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const Run run = find_run<Rope, S::kThreads>(a, per_row, S::kWarps, cta, gridDim.x);
  auto clear = [&]() {     // rows with nothing to attend to
    for (int m = cta; m < a.rows; m += gridDim.x) {
      bool beyond;
      if (extent_of<Rope>(a, m, beyond).tiles != 0) continue;
      uint4* out = reinterpret_cast<uint4*>(static_cast<T*>(a.out) + int64_t(m) * a.q_heads * D);
      for (int i = threadIdx.x; i < a.q_heads * D / 8; i += S::kThreads) out[i] = make_uint4(0u, 0u, 0u, 0u);
    }
  };
  if (run.begin >= run.end) {
    clear();
    return;
  }

  uint8_t* ring = smem + S::kRing + warp * S::kStages * S::kStageBytes;
  uint32_t* valid_s = reinterpret_cast<uint32_t*>(smem + S::kValid) + warp * S::kStages;
  const int own = run.end - run.begin;
  const int mine = own > warp ? (own - warp + S::kWarps - 1) / S::kWarps : 0;   // tiles of this warp

  // ---- copies: the page of a tile is looked up one tile before its copies are issued
  Cursor<Rope> ahead(a, run);
  struct Page {
    uint32_t id, inner;     // of lane % 16, the slot of a tile: its page, and the 16-byte vectors behind the page's beginning
    bool inside;
  };
  int looked_up = 0;
  auto look_up = [&]() {
    Page page{0u, 0u, false};
    if (looked_up >= mine) return page;
    ahead.advance(a, per_row, looked_up == 0 ? warp : S::kWarps);
    ++looked_up;
    const uint32_t slot = uint32_t(ahead.tile) * kTile + (lane & 15);
    page.inside = slot < uint32_t(ahead.extent.held);
    if (page.inside) {
      const uint32_t column = a.layout.page.quotient(slot);
      page.id = uint32_t(__ldg(a.layout.tables + int64_t(ahead.row) * a.layout.table_stride + column));
      page.inner = a.by_head_tiles.quotient(ahead.head) * a.layout.head_stride + (slot - column * a.layout.page.divisor) * a.layout.slot_stride;
    }
    return page;
  };
  int issued = 0, into = 0;
  const uint32_t copies_to = shared_address(ring);
  auto issue = [&](const Page& page) {
    if (issued < mine) {
      uint32_t offset = kNoSlot;
      if (page.inside) {
        if (page.id < a.layout.pages) offset = page.id * a.layout.page_stride + page.inner;
        else atomicOr(&g_paged_attention_status, 1u);
      }
      const uint32_t to = copies_to + into * S::kStageBytes;
      const uint32_t counts = __ballot_sync(0xffffffffu, offset != kNoSlot) & 0xffffu;
      if (lane == 0) valid_s[into] = counts;
      into = into + 1 == S::kStages ? 0 : into + 1;
      if (counts == 0xffffu) {
#pragma unroll
        for (int i = 0; i < S::kOps; ++i) {
          const int row = (i * 32 + lane) / S::kPieces, piece = (i * 32 + lane) % S::kPieces;
          const uint32_t from = __shfl_sync(0xffffffffu, offset, row);
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + S::key_at(row, piece)), "l"(a.k_pages + piece + from) : "memory");
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + S::value_at(row, piece)), "l"(a.v_pages + piece + from) : "memory");
        }
      } else {
        // a slot that does not count is filled with zeros: whatever lies there, a NaN too, stays out of the products
#pragma unroll
        for (int i = 0; i < S::kOps; ++i) {
          const int row = (i * 32 + lane) / S::kPieces, piece = (i * 32 + lane) % S::kPieces;
          const uint32_t from = __shfl_sync(0xffffffffu, offset, row), size = from != kNoSlot ? 16u : 0u;
          const int64_t source = int64_t(size ? from : 0u) + piece;       // not read where nothing is copied
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + S::key_at(row, piece)), "l"(a.k_pages + source), "r"(size) : "memory");
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + S::value_at(row, piece)), "l"(a.v_pages + source), "r"(size) : "memory");
        }
      }
      ++issued;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  Page pages[S::kStages - 1];
#pragma unroll
  for (int i = 0; i < S::kStages - 1; ++i) pages[i] = look_up();

  // ---- the run, item by item.  What an item's beginning reads is fetched while the item before ends.
  Cursor<Rope> at(a, run);
  int done = run.begin, count, position = 0;
  uint4 query_raw[D / 32], new_low, new_high, new_value;
  uint32_t new_slot = kNoSlot;
  auto fetch = [&]() {
    count = min(at.extent.tiles - at.tile, run.end - done);
    const int kv = int(a.by_head_tiles.quotient(at.head)), first = (at.head - kv * a.head_tiles) * kHeads;
    const T* source = static_cast<const T*>(a.q) + int64_t(at.row) * a.q_row;
    const uint4* q = reinterpret_cast<const uint4*>(source + int64_t(kv * a.group + first + g) * a.q_head) + t;
#pragma unroll
    for (int j = 0; j < D / 32; ++j) query_raw[j] = g < a.group - first ? __ldg(q + 4 * j) : make_uint4(0u, 0u, 0u, 0u);
    if constexpr (Rope) {
      position = __ldg(a.positions + at.row);
      // the warp that has the tile of the new token
      if (at.extent.added && at.tile + count == at.extent.tiles && (done - run.begin + count - 1) % S::kWarps == warp) {
        const uint4* k = reinterpret_cast<const uint4*>(source + int64_t(a.q_heads + kv) * D);
        const uint4* v = reinterpret_cast<const uint4*>(source + int64_t(a.q_heads + a.kv_heads + kv) * D);
        if (lane < S::kPieces / 2) { new_low = __ldg(k + lane); new_high = __ldg(k + lane + S::kPieces / 2); }
        if (lane < S::kPieces) new_value = __ldg(v + lane);
        new_slot = a.layout.vector_of(a.layout.tables + int64_t(at.row) * a.layout.table_stride, kv, at.extent.held);
      }
    }
  };
  fetch();
#pragma unroll
  for (int i = 0; i < S::kStages - 1; ++i) issue(pages[i]);
  Page next = look_up();
  clear();

  // where a lane's pieces lie in a stage: of the keys 32j .. and 32j + 32 .. (j even) of row g, of the values of row 2t
  const int key0 = S::key_at(g, t), key1 = S::key_at(g, t + 4), value0 = S::value_at(2 * t, g);
  int turned = -1, stage = 0;
  bool exact = false;
  for (;;) {
    const int kv = int(a.by_head_tiles.quotient(at.head)), first = (at.head - kv * a.head_tiles) * kHeads;
    const int head0 = kv * a.group + first, heads = min(kHeads, a.group - first);
    // The new key is turned in 64 bits: it is kept, and rounded once.  Where this run does not hold it, the queries' rotation
    // does with 32.
    const bool ends = Rope && at.extent.added && at.tile + count == at.extent.tiles;
    if (Rope && (turned != at.row || (ends && !exact))) {
      turned = at.row;
      exact = ends;
      for (int i = threadIdx.x; i < D / 2; i += S::kThreads) {
        double turns = double(position) * turns_s[i];
        turns -= rint(turns);
        float sine, cosine;
        if (ends) {
          double2 both;
          sincospi(2. * turns, &both.y, &both.x);
          exact_s[i] = both;
          cosine = float(both.x);
          sine = float(both.y);
        } else {
          sincospif(2.f * float(turns), &sine, &cosine);
        }
        cosine_s[i] = make_float2(cosine * Y::kRotated, sine * Y::kRotated);
      }
      __syncthreads();
    }
    // rotates pieces of 8 dimensions d.. and d + D/2.. of a query, times kRotated
    auto rotate = [&](const uint4& low, const uint4& high, int d, float (&x)[8], float (&y)[8]) {
      const uint32_t l[4] = {low.x, low.y, low.z, low.w}, h[4] = {high.x, high.y, high.z, high.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 p = Y::widen(l[i]), q = Y::widen(h[i]), c0 = cosine_s[d + 2 * i], c1 = cosine_s[d + 2 * i + 1];
        x[2 * i] = p.x * c0.x - q.x * c0.y;
        x[2 * i + 1] = p.y * c1.x - q.y * c1.y;
        y[2 * i] = q.x * c0.x + p.x * c0.y;
        y[2 * i + 1] = q.y * c1.x + p.y * c1.y;
      }
    };
    // queries: head g, dimensions 32j + 8t ..
    uint32_t query[D / 32][4], rest[Rope ? D / 32 : 1][4];
    uint4* third_s = reinterpret_cast<uint4*>(smem + S::kThird) + warp * D + lane;
    {
      if constexpr (Rope) {
#pragma unroll
        for (int j = 0; j < D / 64; ++j) {
          float x[8], y[8];
          rotate(query_raw[j], query_raw[j + D / 64], 32 * j + 8 * t, x, y);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            split<T>(x[2 * i], x[2 * i + 1], query[j][i], rest[j][i]);
            split<T>(y[2 * i], y[2 * i + 1], query[j + D / 64][i], rest[j + D / 64][i]);
          }
          if constexpr (Weighted) {
            auto left = [](uint32_t pair, uint32_t rest, float lo, float hi) {
              const float2 a = Y::widen(pair), b = Y::widen(rest);
              return Y::narrow(lo - a.x - b.x, hi - a.y - b.y);
            };
            const int k = j + D / 64;
            third_s[j * 32] = make_uint4(left(query[j][0], rest[j][0], x[0], x[1]), left(query[j][1], rest[j][1], x[2], x[3]),
                                         left(query[j][2], rest[j][2], x[4], x[5]), left(query[j][3], rest[j][3], x[6], x[7]));
            third_s[k * 32] = make_uint4(left(query[k][0], rest[k][0], y[0], y[1]), left(query[k][1], rest[k][1], y[2], y[3]),
                                         left(query[k][2], rest[k][2], y[4], y[5]), left(query[k][3], rest[k][3], y[6], y[7]));
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {
          query[j][0] = query_raw[j].x; query[j][1] = query_raw[j].y; query[j][2] = query_raw[j].z; query[j][3] = query_raw[j].w;
        }
      }
    }
    float out[D / 16][4];   // [64j.. : 4j + i]: dimensions 64j + 8g + 2i (0, 1) and + 1 (2, 3) of heads 2t and 2t + 1
#pragma unroll
    for (int i = 0; i < D / 16; ++i) out[i][0] = out[i][1] = out[i][2] = out[i][3] = 0.f;
    float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};

    const int skip = (done - run.begin) % S::kWarps;
    for (int i = warp >= skip ? warp - skip : warp - skip + S::kWarps; i < count; i += S::kWarps) {
      asm volatile("cp.async.wait_group %0;" ::"n"(S::kStages - 2) : "memory");
      __syncwarp();   // every lane's copies of this tile are there, and every lane has read the tile before
      issue(next);    // into the stage of the tile before
      next = look_up();
      uint8_t* from = ring + stage * S::kStageBytes;
      uint32_t valid = valid_s[stage];
      stage = stage + 1 == S::kStages ? 0 : stage + 1;
      const int tile = at.tile + i;
      if (Rope && at.extent.added && tile == at.extent.held / kTile) {
        // the token that this call adds goes into the ring, and into the cache
        const int r = at.extent.held % kTile;
        if (new_slot == kNoSlot) {
          if (lane == 0) atomicOr(&g_paged_attention_status, 1u);
        } else {
          const bool store = first == 0;
          if (lane < S::kPieces / 2) {
            float x[8], y[8];
            const uint32_t l[4] = {new_low.x, new_low.y, new_low.z, new_low.w}, h[4] = {new_high.x, new_high.y, new_high.z, new_high.w};
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float2 ps = Y::widen(l[e >> 1]), qs = Y::widen(h[e >> 1]);
              const double p = e & 1 ? ps.y : ps.x, q = e & 1 ? qs.y : qs.x;
              const double2 turn = exact_s[8 * lane + e];
              x[e] = float(p * turn.x - q * turn.y);
              y[e] = float(q * turn.x + p * turn.y);
            }
            const uint4 low = make_uint4(Y::narrow(x[0], x[1]), Y::narrow(x[2], x[3]), Y::narrow(x[4], x[5]), Y::narrow(x[6], x[7]));
            const uint4 high = make_uint4(Y::narrow(y[0], y[1]), Y::narrow(y[2], y[3]), Y::narrow(y[4], y[5]), Y::narrow(y[6], y[7]));
            *reinterpret_cast<uint4*>(from + S::key_at(r, lane)) = low;
            *reinterpret_cast<uint4*>(from + S::key_at(r, lane + S::kPieces / 2)) = high;
            if (store) {
              a.k_pages[int64_t(new_slot) + lane] = low;
              a.k_pages[int64_t(new_slot) + lane + S::kPieces / 2] = high;
            }
          }
          if (lane < S::kPieces) {
            *reinterpret_cast<uint4*>(from + S::value_at(r, lane)) = new_value;
            if (store) a.v_pages[int64_t(new_slot) + lane] = new_value;
          }
          valid |= 1u << r;
        }
        __syncwarp();
      }
      // scores of slots g (0, 1) and g + 8 (2, 3) for heads 2t and 2t + 1
      float score[4] = {0.f, 0.f, 0.f, 0.f}, small[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < D / 32; ++j) {
        const uint8_t* key = from + (j & 1 ? key1 : key0) + (j >> 1) * 128;
        const uint4 x = *reinterpret_cast<const uint4*>(key), y = *reinterpret_cast<const uint4*>(key + 8 * S::kPieces * 16);
        Y::mma(score, x.x, y.x, x.y, y.y, query[j][0], query[j][1]);
        Y::mma(Rope ? score : small, x.z, y.z, x.w, y.w, query[j][2], query[j][3]);
        if constexpr (Rope) {
          Y::mma(small, x.x, y.x, x.y, y.y, rest[j][0], rest[j][1]);
          Y::mma(small, x.z, y.z, x.w, y.w, rest[j][2], rest[j][3]);
          if constexpr (Weighted) {
            const uint4 third = third_s[j * 32];
            Y::mma(small, x.x, y.x, x.y, y.y, third.x, third.y);
            Y::mma(small, x.z, y.z, x.w, y.w, third.z, third.w);
          }
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) score[e] = (score[e] + small[e]) * a.scale_log2;
      if (valid != 0xffffu) {
        valid >>= g;
#pragma unroll
        for (int e = 0; e < 4; ++e) score[e] = valid >> (e >> 1) * 8 & 1u ? score[e] : -INFINITY;
      }
      if (a.weights != nullptr) {
        float* to = a.scores + int64_t(done + i) * (min(a.group, kHeads) * kTile);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (2 * t + (e & 1) < heads) to[(2 * t + (e & 1)) * kTile + g + (e >> 1) * 8] = score[e];
      }
      float high[2] = {fmaxf(score[0], score[2]), fmaxf(score[1], score[3])};
#pragma unroll
      for (int step = 4; step < 32; step <<= 1) {
        high[0] = fmaxf(high[0], __shfl_xor_sync(0xffffffffu, high[0], step));
        high[1] = fmaxf(high[1], __shfl_xor_sync(0xffffffffu, high[1], step));
      }
      if (__any_sync(0xffffffffu, high[0] > top[0] || high[1] > top[1])) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float now = fmaxf(top[c], high[c]);
          const float fade = now > -INFINITY ? power_of_two(top[c] - now) : 1.f;
          top[c] = now;
          sum[c] *= fade;
#pragma unroll
          for (int k = 0; k < D / 16; ++k) { out[k][c] *= fade; out[k][c + 2] *= fade; }
        }
      }
      const float base[2] = {top[0] > -INFINITY ? top[0] - kShift : 0.f, top[1] > -INFINITY ? top[1] - kShift : 0.f};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        score[e] = power_of_two(score[e] - base[e & 1]);
        sum[e & 1] += score[e];
      }
      uint32_t p0, p1, r0, r1;
      split<T>(score[0], score[1], p0, r0);
      split<T>(score[2], score[3], p1, r1);
      p0 = turn_matrix(p0); p1 = turn_matrix(p1); r0 = turn_matrix(r0); r1 = turn_matrix(r1);
#pragma unroll
      for (int j = 0; j < D / 64; ++j) {
        uint4 v[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = *reinterpret_cast<const uint4*>(from + value0 + ((r & 1) + (r >> 1) * 8) * (S::kPieces * 16) + j * 128);
        const uint32_t words[4][4] = {{v[0].x, v[0].y, v[0].z, v[0].w}, {v[1].x, v[1].y, v[1].z, v[1].w},
                                      {v[2].x, v[2].y, v[2].z, v[2].w}, {v[3].x, v[3].y, v[3].z, v[3].w}};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t a0 = __byte_perm(words[0][k], words[1][k], 0x5410), a1 = __byte_perm(words[0][k], words[1][k], 0x7632);
          const uint32_t a2 = __byte_perm(words[2][k], words[3][k], 0x5410), a3 = __byte_perm(words[2][k], words[3][k], 0x7632);
          Y::mma(out[4 * j + k], a0, a1, a2, a3, p0, p1);
          Y::mma(out[4 * j + k], a0, a1, a2, a3, r0, r1);
        }
      }
    }

    // ---- the warps meet, each in the stage of its ring that no copy is under way to
#pragma unroll
    for (int step = 4; step < 32; step <<= 1) {
      sum[0] += __shfl_xor_sync(0xffffffffu, sum[0], step);
      sum[1] += __shfl_xor_sync(0xffffffffu, sum[1], step);
    }
    const int free_stage = stage == 0 ? S::kStages - 1 : stage - 1;
    float* out_s = reinterpret_cast<float*>(ring + free_stage * S::kStageBytes);
    float2* norm_s = reinterpret_cast<float2*>(smem + S::kNorm);
    int* meet_s = reinterpret_cast<int*>(smem + S::kMeet);
    if (lane == 0) meet_s[warp] = S::kRing + (warp * S::kStages + free_stage) * S::kStageBytes;
    __syncwarp();
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int head = 2 * t + c;
      if (g == 0) norm_s[warp * kHeads + head] = make_float2(top[c], sum[c]);
      float* row = out_s + head * S::kRowFloats + 8 * g;
#pragma unroll
      for (int j = 0; j < D / 64; ++j) {
        *reinterpret_cast<float4*>(row + 64 * j) = make_float4(out[4 * j][c], out[4 * j][c + 2], out[4 * j + 1][c], out[4 * j + 1][c + 2]);
        *reinterpret_cast<float4*>(row + 64 * j + 4) = make_float4(out[4 * j + 2][c], out[4 * j + 2][c + 2], out[4 * j + 3][c], out[4 * j + 3][c + 2]);
      }
    }
    const bool from_start = at.tile == 0, whole = from_start && count == at.extent.tiles;
    const int begin = done - at.tile, end = begin + at.extent.tiles;          // of the item
    const int64_t out_row = int64_t(at.row) * a.q_heads + head0;
    done += count;
    const bool more = done < run.end;
    if (more) {
      at.advance(a, per_row, count);
      fetch();
    }
    __syncthreads();
    for (int index = threadIdx.x; index < heads * (D / 8); index += S::kThreads) {
      const int head = index / (D / 8), d = (index - head * (D / 8)) * 8;
      float all = -INFINITY, total = 0.f, x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < S::kWarps; ++w) all = fmaxf(all, norm_s[w * kHeads + head].x);
#pragma unroll
      for (int w = 0; w < S::kWarps; ++w) {
        const float2 norm = norm_s[w * kHeads + head];
        if (norm.y == 0.f) continue;            // no tiles, or none whose slots count
        const float fade = power_of_two(norm.x - all);
        total += norm.y * fade;
        const float4* row = reinterpret_cast<const float4*>(smem + meet_s[w] + (head * S::kRowFloats + d) * 4);
        const float4 lo = row[0], hi = row[1];
        x[0] += lo.x * fade; x[1] += lo.y * fade; x[2] += lo.z * fade; x[3] += lo.w * fade;
        x[4] += hi.x * fade; x[5] += hi.y * fade; x[6] += hi.z * fade; x[7] += hi.w * fade;
      }
      if (whole) {
        const float inverse = total == 0.f ? 0.f : 1.f / total;
        *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + (out_row + head) * D + d) =
            make_uint4(Y::narrow(x[0] * inverse, x[1] * inverse), Y::narrow(x[2] * inverse, x[3] * inverse),
                       Y::narrow(x[4] * inverse, x[5] * inverse), Y::narrow(x[6] * inverse, x[7] * inverse));
        if (a.weights != nullptr && d == 0) a.norm[out_row + head] = all - kShift + log2f(total);
      } else {
        const int64_t slot = (int64_t(cta) * 2 + from_start) * kHeads + head;
        float4* row = reinterpret_cast<float4*>(a.partial + slot * D + d);
        row[0] = make_float4(x[0], x[1], x[2], x[3]);
        row[1] = make_float4(x[4], x[5], x[6], x[7]);
        if (d == 0) a.partial_norm[slot] = make_float2(all, total);
      }
    }
    if (!whole) {
      const int left = run.holder(begin), parts = run.holder(end - 1) - left + 1;      // the CTAs that the item lies in
      const int first = (cta - left) / kGroup * kGroup, members = min(kGroup, parts - first);
      unsigned int* ticket_s = reinterpret_cast<unsigned int*>(smem + S::kTicket);
      if (last_of(a.tickets + (left + first) * 3 + (first == 0), members, ticket_s)) {
        const bool final = parts <= kGroup;
        join<T, D, S::kThreads>(a, left, first, 1, members, heads, out_row, final, norm_s);
        if (!final && last_of(a.tickets + left * 3 + 2, (parts + kGroup - 1) / kGroup, ticket_s))
          join<T, D, S::kThreads>(a, left, 0, kGroup, (parts + kGroup - 1) / kGroup, heads, out_row, true, norm_s);
      }
    }
    if (!more) break;
    __syncthreads();
  }
}

// acc[slot] += the weights of the group's heads, from the scores that the first launch left.  A half warp per tile of 16
// slots; the heads are added in their order.
constexpr int kWeightThreads = 256;

template <bool Rope>
__global__ void __launch_bounds__(kWeightThreads) paged_weight_kernel(AttentionArguments a) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  // lengths, tables and weights are there: the kernel before lets this one begin only after its own wait
  constexpr int kParts = kWeightThreads / kTile;
  const Run run = find_run<Rope, kWeightThreads, true>(a, a.kv_heads, kParts, blockIdx.x, gridDim.x);
  const bool idle = threadIdx.x / kTile >= run.end - run.begin;
  if (idle) asm volatile("griddepcontrol.wait;" ::: "memory");
  if (idle) return;
  const int part = threadIdx.x / kTile, lane = threadIdx.x % kTile, stored = min(a.group, kHeads);
  Cursor<Rope, true> at(a, run);
  int before = run.begin - (at.head * at.extent.tiles + at.tile);      // tiles of the rows before
  int row = at.row;
  at.advance(a, a.kv_heads, part);
  auto catch_up = [&]() {
    for (; row < at.row; ++row) {
      bool beyond;
      before += extent_of<Rope, true>(a, row, beyond).tiles * a.kv_heads;
    }
  };
  bool waited = false;
  for (int done = run.begin + part;;) {
    catch_up();
    const int slot = at.tile * kTile + lane;
    const int* table = a.layout.tables + int64_t(at.row) * a.layout.table_stride;
    const int64_t to = slot < at.extent.held + at.extent.added ? a.layout.weight_of<true>(table, a.kv_heads, at.head, slot) : -1;
    // the slot of a new token begins at zero; the kernel before writes no weights
    const float held = to >= 0 && slot != at.extent.held ? __ldcg(a.weights + to) : 0.f;
    if (!waited) asm volatile("griddepcontrol.wait;" ::: "memory");
    waited = true;
    if (to >= 0) {
      float total = 0.f;
      for (int tile = 0; tile < a.head_tiles; ++tile) {
        // the scores lie in the order of the first launch: (row, head, head tile, tile)
        const int64_t from = before * a.head_tiles + (at.head * a.head_tiles + tile) * at.extent.tiles + at.tile;
        const int heads = min(kHeads, a.group - tile * kHeads);
        const float* norm = a.norm + int64_t(at.row) * a.q_heads + at.head * a.group + tile * kHeads;
#pragma unroll
        for (int h = 0; h < kHeads; ++h) total += h < heads ? power_of_two(a.scores[(from * stored + h) * kTile + lane] - norm[h]) : 0.f;
      }
      a.weights[to] = held + total;
    }
    done += kParts;
    if (done >= run.end) break;
    at.advance(a, a.kv_heads, kParts);
  }
}

int64_t aligned(int64_t bytes) { return (bytes + 255) / 256 * 256; }

// CTAs of the first launch, and where the parts of its workspace begin.
struct Workspace {
  int ctas;
  int64_t partial, partial_norm, norm, scores, bytes;
  Workspace(int rows, int q_heads, int kv_heads, int head_dim, int page, int columns, bool weights) {
    ctas = device_info().sm_count * ctas_of(head_dim, false);
    const int group = q_heads / kv_heads, head_tiles = (group + kHeads - 1) / kHeads;
    if (ctas > MKB_PAGED_STATE_BYTES / 12) ctas = MKB_PAGED_STATE_BYTES / 12;      // three tickets each
    partial = 0;
    partial_norm = partial + aligned(int64_t(ctas) * 2 * kHeads * head_dim * 4);
    norm = partial_norm + aligned(int64_t(ctas) * 2 * kHeads * 8);
    scores = norm + (weights ? aligned(int64_t(rows) * q_heads * 4) : 0);
    const int64_t tiles = int64_t(rows) * kv_heads * head_tiles * ((int64_t(columns) * page + kTile - 1) / kTile);
    bytes = scores + (weights ? aligned(tiles * (group < kHeads ? group : kHeads) * kTile * 4) : 0);
  }
};

template <typename T, int D, bool Rope, bool Weighted>
int launch(AttentionArguments& a, void* stream) {
  using S = Shape<D, Rope, Weighted>;
  int device = 0;
  cudaGetDevice(&device);
  static std::atomic<uint64_t> opted{0};
  if (!(opted.load(std::memory_order_acquire) >> (device & 63) & 1)) {
    const cudaError_t set = cudaFuncSetAttribute(paged_attention_kernel<T, D, Rope, Weighted>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes);
    if (set != cudaSuccess) return cuda_fail(set, "paged attention shared memory");
    opted.fetch_or(uint64_t(1) << (device & 63), std::memory_order_release);
  }
  a.ctas = min(a.ctas, device_info().sm_count * S::kCtas);
  if (Rope) a.scale_log2 /= Types<T>::kRotated;
  cudaError_t launched = launch_dependent(paged_attention_kernel<T, D, Rope, Weighted>, dim3(a.ctas), dim3(S::kThreads), S::kBytes, stream, a);
  if (launched == cudaSuccess && a.weights != nullptr)
    launched = launch_dependent(paged_weight_kernel<Rope>, dim3(a.ctas * 2), dim3(kWeightThreads), 0, stream, a);
  if (launched != cudaSuccess) return cuda_fail(launched, "paged attention launch");
  return MKB_OK;
}

template <typename T, bool Rope, bool Weighted = false>
int dispatch(AttentionArguments& a, int head_dim, void* stream) {
  switch (head_dim) {
    case 64: return launch<T, 64, Rope, Weighted>(a, stream);
    case 128: return launch<T, 128, Rope, Weighted>(a, stream);
    case 192: return launch<T, 192, Rope, Weighted>(a, stream);
    default: return launch<T, 256, Rope, Weighted>(a, stream);
  }
}

// Checks what both entry points share, fills the rest of `a` and launches.
int attend(const char* what, AttentionArguments& a, bool rope, void* out, float* weights, int M, int q_heads, int kv_heads, int head_dim,
           int page, int columns, float scale, int dtype, void* state, void* workspace, int64_t workspace_bytes, void* stream) {
  MKB_REQUIRE(a.q && a.lengths && out && (a.positions || !rope), MKB_E_ARGUMENT, "%s: null pointer", what);
  MKB_REQUIRE(q_heads > 0 && q_heads % kv_heads == 0, MKB_E_ARGUMENT, "%s: %d query heads for %d key-value heads", what, q_heads, kv_heads);
  MKB_REQUIRE(dtype == MKB_F16 || dtype == MKB_BF16, MKB_E_UNSUPPORTED, "%s: dtype tag %d (fp16 and bf16 supported)", what, dtype);
  MKB_REQUIRE(M <= 65535 && q_heads <= 65535, MKB_E_UNSUPPORTED, "%s: %d sequences of %d heads", what, M, q_heads);
  MKB_REQUIRE(fabsf(scale) < INFINITY, MKB_E_ARGUMENT, "%s: scale is not finite", what);
  MKB_REQUIRE(((reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(out)) & 15) == 0 && a.q_row % 8 == 0 && a.q_head % 8 == 0,
              MKB_E_ALIGNMENT, "%s: queries and outputs lie on 16-byte vectors", what);
  MKB_REQUIRE(int64_t(M) * kv_heads * ((q_heads / kv_heads + kHeads - 1) / kHeads) * ((int64_t(columns) * page + kTile - 1) / kTile) < (int64_t(1) << 31),
              MKB_E_UNSUPPORTED, "%s: %d sequences of %d pages of %d slots", what, M, columns, page);
  const int64_t out_row = int64_t(q_heads) * head_dim, q_width = rope ? (int64_t(q_heads) + 2 * kv_heads) * head_dim : (q_heads - 1) * a.q_head + head_dim;
  const bool in_place = !rope && out == a.q && a.q_head == head_dim && (M == 1 || a.q_row == out_row);
  MKB_REQUIRE(a.q_row >= 0 && a.q_head >= 0, MKB_E_ARGUMENT, "%s: negative stride", what);
  MKB_REQUIRE(in_place || !overlap(a.q, ((M - 1) * a.q_row + q_width) * 2, out, M * out_row * 2), MKB_E_ARGUMENT,
              "%s: the output overlaps the queries", what);
  const Workspace parts(M, q_heads, kv_heads, head_dim, page, columns, weights != nullptr);
  MKB_REQUIRE(workspace != nullptr && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0 && workspace_bytes >= parts.bytes, MKB_E_ARGUMENT,
              "%s: workspace of %lld bytes, %lld needed", what, (long long)workspace_bytes, (long long)parts.bytes);
  MKB_REQUIRE(state != nullptr && (reinterpret_cast<uintptr_t>(state) & 3) == 0, MKB_E_ARGUMENT, "%s: no state", what);
  char* base = static_cast<char*>(workspace);
  a.out = out; a.weights = weights; a.rows = M; a.q_heads = q_heads; a.kv_heads = kv_heads; a.group = q_heads / kv_heads;
  a.head_tiles = (a.group + kHeads - 1) / kHeads; a.by_head_tiles = FastDivide::of(uint32_t(a.head_tiles)); a.ctas = parts.ctas;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.partial = reinterpret_cast<float*>(base + parts.partial);
  a.partial_norm = reinterpret_cast<float2*>(base + parts.partial_norm);
  a.tickets = static_cast<unsigned int*>(state);
  a.norm = reinterpret_cast<float*>(base + parts.norm);
  a.scores = reinterpret_cast<float*>(base + parts.scores);
  if (dtype == MKB_F16) return rope ? dispatch<__half, true>(a, head_dim, stream) : dispatch<__half, false>(a, head_dim, stream);
  if (rope && weights != nullptr) return dispatch<__nv_bfloat16, true, true>(a, head_dim, stream);
  return rope ? dispatch<__nv_bfloat16, true>(a, head_dim, stream) : dispatch<__nv_bfloat16, false>(a, head_dim, stream);
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
  if (M <= 0 || q_heads <= 0 || kv_heads <= 0 || q_heads < kv_heads || head_dim <= 0 || page <= 0 || columns <= 0) return 0;
  return mkb::Workspace(M, q_heads, kv_heads, head_dim, page, columns, with_weights != 0).bytes;
}

extern "C" int mkb_paged_attention_decode(const void* q, const int* lengths, const void* k_pages, const void* v_pages,
                                          const int* tables, void* out, float* weights, int M, int q_heads, int kv_heads,
                                          int head_dim, int page, int columns, int64_t pages, int64_t page_stride,
                                          int64_t head_stride, int64_t slot_stride, int64_t table_stride, int64_t q_row_stride,
                                          int64_t q_head_stride, float scale, int dtype, void* state, void* workspace,
                                          int64_t workspace_bytes, void* stream) {
  using namespace mkb;
  const char* what = "paged_attention_decode";
  MKB_REQUIRE(M >= 0, MKB_E_ARGUMENT, "%s: bad shape", what);
  if (M == 0) return MKB_OK;
  AttentionArguments a{};
  const int status = paged_layout(&a.layout, what, k_pages, v_pages, tables, kv_heads, head_dim, page, columns, pages, page_stride,
                                  head_stride, slot_stride, table_stride);
  if (status != MKB_OK) return status;
  a.q = q; a.lengths = lengths; a.q_row = q_row_stride; a.q_head = q_head_stride;
  a.k_pages = static_cast<uint4*>(const_cast<void*>(k_pages)); a.v_pages = static_cast<uint4*>(const_cast<void*>(v_pages));
  return attend(what, a, false, out, weights, M, q_heads, kv_heads, head_dim, page, columns, scale, dtype, state, workspace, workspace_bytes, stream);
}

extern "C" int mkb_paged_rope_attention_decode(const void* qkv, const int* positions, const int* lengths, void* k_pages, void* v_pages,
                                               const int* tables, void* out, float* weights, int M, int q_heads, int kv_heads,
                                               int head_dim, int page, int columns, int64_t pages, int64_t page_stride,
                                               int64_t head_stride, int64_t slot_stride, int64_t table_stride, int64_t qkv_row_stride,
                                               float theta, float scale, int dtype, void* state, void* workspace,
                                               int64_t workspace_bytes, void* stream) {
  using namespace mkb;
  const char* what = "paged_rope_attention_decode";
  MKB_REQUIRE(M >= 0, MKB_E_ARGUMENT, "%s: bad shape", what);
  if (M == 0) return MKB_OK;
  AttentionArguments a{};
  const int status = paged_layout(&a.layout, what, k_pages, v_pages, tables, kv_heads, head_dim, page, columns, pages, page_stride,
                                  head_stride, slot_stride, table_stride);
  if (status != MKB_OK) return status;
  MKB_REQUIRE(theta > 0.f && theta < INFINITY, MKB_E_ARGUMENT, "%s: theta is not positive", what);
  a.q = qkv; a.positions = positions; a.lengths = lengths; a.q_row = qkv_row_stride; a.q_head = head_dim; a.theta = theta;
  a.k_pages = static_cast<uint4*>(k_pages); a.v_pages = static_cast<uint4*>(v_pages);
  return attend(what, a, true, out, weights, M, q_heads, kv_heads, head_dim, page, columns, scale, dtype, state, workspace, workspace_bytes, stream);
}
