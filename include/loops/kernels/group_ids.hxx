/**
 * @file group_ids.hxx
 * @brief Groups positions by id: a stable sort of (id, position), which is the COO -> CSC conversion of a matrix with one nonzero per
 * position (row = position, column = id).  What the embedding gradient sums over and what experts' products are dispatched by.
 *
 * key(i) = id_i - first for ids in [first, first + rows) other than `drop`, `rows` otherwise (those end up behind the last group).
 *
 *   n <= 8 192   RANK, one launch: an item's place is the number of items that come before it.  Every workgroup holds all keys in LDS and
 *                finds the places of 16 items: n^2 comparisons over the whole chip, whatever the ids.
 *   beyond       least-significant-digit radix sort, digits of at most 10 bits, ceil(log2(rows + 1) / digits) of them, two launches each.
 *                COUNT: workgroup w counts the digits of its span (n / W consecutive items, W <= 128).  PLACE: every workgroup adds up the
 *                counts of the spans before it (W x digits words from L2; no scan launch), then each of its 16 wavefronts counts and
 *                places its own sixteenth of the span.
 *
 * A wavefront ranks 64 items at a time without atomics: one ballot per digit bit leaves each lane the mask of the lanes with its digit;
 * the rank is the number of mask bits below the lane and the last of them advances the wavefront's counter in LDS.  Items are taken in
 * order, so equal ids keep the order of their positions and the result is the same in every run.
 *
 * Few items are a matter of launches and of the latency of their dependent steps: 2 048 positions take 3.7 us by RANK (7.5 by one pass of
 * the sort, 14.2 by two), 8 192 8.9 (8.3, 15.4), 16 384 26 (8.4, 16).  524 288 positions of 9 bits take 16 us in two launches, 131 072 of 18 bits
 * 25 in four; more or fewer spans (64, 256) and holding the items in registers between counting and placing changed neither.
 */
#pragma once

#include <cstddef>
#include <cstdint>
#include <type_traits>

#include <hip/hip_runtime.h>

#include <loops/util/wave.hxx>

namespace loops {
namespace kernels {
namespace group_ids {

constexpr int threads = 1024;
constexpr int waves = threads / wave::size;
constexpr int max_digit_bits = 10;
constexpr int max_digits = 1 << max_digit_bits;
constexpr int rank_items = 8192;  ///< most items of the RANK form
constexpr int max_spans = 128;

/// Which ids count, and what they become.
struct key_map {
  long long first;
  long long drop;  ///< id left out (negative: none)
  int rows;
  template <typename id_t>
  __device__ __forceinline__ unsigned int operator()(id_t id) const {
    const long long v = static_cast<long long>(id);
    const unsigned long long at = static_cast<unsigned long long>(v) - static_cast<unsigned long long>(first);
    return at < static_cast<unsigned long long>(rows) && v != drop ? static_cast<unsigned int>(at) : static_cast<unsigned int>(rows);
  }
};

struct item_t {
  unsigned int key;
  int position;
};

struct plan_t {
  int passes;  ///< 0: RANK
  int bits;    ///< per digit
  int spans;   ///< workgroups of a launch
  int span;    ///< items per workgroup
};

/// Bits are shared out evenly: 18 bits are two digits of 9.  A span is 1 024 items (one per thread) until there would be more than 128.
inline plan_t plan_for(int n, int rows) {
  plan_t p{0, 0, 0, 0};
  if (n <= rank_items) return p;
  int bits = 2;
  while (bits < 31 && (static_cast<unsigned int>(rows) >> bits) != 0u) ++bits;
  p.passes = (bits + max_digit_bits - 1) / max_digit_bits;
  p.bits = (bits + p.passes - 1) / p.passes;
  const int want = (n + threads - 1) / threads;
  const int w = want < max_spans ? want : max_spans;
  const long long per = (static_cast<long long>(n) + w - 1) / w;
  p.span = static_cast<int>((per + threads - 1) / threads * threads);
  p.spans = static_cast<int>((static_cast<long long>(n) + p.span - 1) / p.span);
  return p;
}

inline std::size_t item_bytes(int n) { return (static_cast<std::size_t>(n) * sizeof(item_t) + 255) & ~static_cast<std::size_t>(255); }

/// Items between the passes (two buffers in turn), counts[spans][digits].
inline std::size_t workspace_bytes(int n, int rows) {
  const plan_t p = plan_for(n, rows);
  if (p.passes == 0) return 0;
  return item_bytes(n) * static_cast<std::size_t>(p.passes > 2 ? 2 : p.passes - 1) +
         static_cast<std::size_t>(p.spans) * (static_cast<std::size_t>(1) << p.bits) * sizeof(int);
}

namespace detail {

/// LDS accesses of ONE wavefront execute in program order; this keeps the compiler to it.
__device__ __forceinline__ void wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

/// Lanes of the wavefront that are `valid` and hold the same digit (0 for lanes that are not valid).
__device__ __forceinline__ unsigned long long same_digit(unsigned int digit, int bits, bool valid) {
  unsigned long long mask = __ballot(valid);
  for (int b = 0; b < bits; ++b) {
    const bool set = (digit >> b) & 1u;
    const unsigned long long with = __ballot(set);
    mask &= set ? with : ~with;
  }
  return valid ? mask : 0ull;
}

__device__ __forceinline__ int lanes_below(unsigned long long mask) {
  return static_cast<int>(__builtin_amdgcn_mbcnt_hi(static_cast<unsigned int>(mask >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<unsigned int>(mask), 0u)));
}

/// Where the lane's item goes among the wavefront's items of its digit: `next[digit]` before the call plus its rank; advances next[].
__device__ __forceinline__ int take(int* __restrict__ next, unsigned int digit, int bits, bool valid) {
  const unsigned long long mask = same_digit(digit, bits, valid);
  const int rank = lanes_below(mask);
  int at = 0;
  if (valid) at = next[digit] + rank;
  wave_order();
  if (valid && rank == __popcll(mask) - 1) next[digit] = at + 1;
  wave_order();
  return at;
}

/// Exclusive prefix sum of one int per thread over the workgroup of 1 024 (`scratch`: 16 ints of LDS).
__device__ __forceinline__ int block_exclusive_sum(int v, int* __restrict__ scratch) {
  const int w = static_cast<int>(threadIdx.x) / wave::size;
  const int inclusive = wave::inclusive_sum(v);
  if (wave::lane() == wave::size - 1) scratch[w] = inclusive;
  __syncthreads();
  int before = 0;
  for (int i = 0; i < w; ++i) before += scratch[i];
  __syncthreads();
  return before + inclusive - v;
}

/// s_count[wave][digit] holds each wavefront's counts: turns them into the place of the wavefront's first item of the digit, `base` =
/// the place of the workgroup's first item of digit threadIdx.x.
__device__ __forceinline__ void places(int* __restrict__ s_count, int digits, int base) {
  const int d = threadIdx.x;
  if (d < digits) {
    int at = base;
#pragma unroll
    for (int w = 0; w < waves; ++w) {
      const int c = s_count[w * digits + d];
      s_count[w * digits + d] = at;
      at += c;
    }
  }
}

}  // namespace detail

constexpr int rank_group = 16;                                 ///< items per workgroup of `rank`
constexpr int rank_parts = threads / rank_group;               ///< threads per item

/// Workgroup b finds the places of items [16 b, 16 b + 16).  Thread (part, item) compares its item with every 64th group of 4 keys, so
/// that a wavefront's LDS read fetches 16 keys for 16 items each.
template <typename id_t>
__global__ void __launch_bounds__(threads)
rank(const int n, const id_t* __restrict__ in, const key_map map, int* __restrict__ ids, int* __restrict__ positions) {
  typedef unsigned int quad_t __attribute__((ext_vector_type(4)));
  __shared__ quad_t s_key[rank_items / 4];
  __shared__ int s_before[waves][rank_group];
  const int tid = threadIdx.x;
  const int quads = (n + 3) / 4;
  unsigned int* const keys = reinterpret_cast<unsigned int*>(s_key);
  for (int i = tid; i < quads * 4; i += threads) keys[i] = i < n ? map(in[i]) : 0xFFFFFFFFu;  // (behind every key)
  __syncthreads();
  const int first = static_cast<int>(blockIdx.x) * rank_group;
  const int mine = first + tid % rank_group;
  const int part = tid / rank_group;
  const unsigned int key = keys[mine < n ? mine : 0];
  int before = 0;
  const int own = first / 4, behind = own + rank_group / 4;
#pragma unroll 4
  for (int q = part; q < own; q += rank_parts) {
    const quad_t k = s_key[q];
    before += (k.x <= key) + (k.y <= key) + (k.z <= key) + (k.w <= key);
  }
#pragma unroll 4
  for (int q = behind + part; q < quads; q += rank_parts) {
    const quad_t k = s_key[q];
    before += (k.x < key) + (k.y < key) + (k.z < key) + (k.w < key);
  }
  if (part < rank_group) {  // the workgroup's own 16: equal keys in the order of their positions
    const int j = first + part;
    if (j < n) before += keys[j] < key || (keys[j] == key && j < mine);
  }
#pragma unroll
  for (int d = rank_group; d < wave::size; d <<= 1) before += __shfl_xor(before, d, wave::size);
  if (wave::lane() < rank_group) s_before[tid / wave::size][wave::lane()] = before;
  __syncthreads();
  if (tid < rank_group && mine < n) {
    int place = 0;
#pragma unroll
    for (int i = 0; i < waves; ++i) place += s_before[i][tid];
    ids[place] = static_cast<int>(key);
    positions[place] = mine;
  }
}

/// Item i of the pass's input: raw ids on the first pass, items afterwards.
template <bool FIRST, typename id_t>
__device__ __forceinline__ item_t read_item(const id_t* __restrict__ raw, const item_t* __restrict__ items, const key_map& map, int i) {
  if constexpr (FIRST) return item_t{map(raw[i]), i};
  else return items[i];
}

template <bool FIRST, typename id_t>
__global__ void __launch_bounds__(threads)
count_digits(const int n, const id_t* __restrict__ raw, const item_t* __restrict__ items, const key_map map, const int shift, const int bits,
             const int span, int* __restrict__ counts) {
  __shared__ int s_count[max_digits];
  const int digits = 1 << bits;
  const int tid = threadIdx.x;
  for (int d = tid; d < digits; d += threads) s_count[d] = 0;
  __syncthreads();
  const int begin = blockIdx.x * span;
  const int end = n - begin < span ? n : begin + span;
  for (int i = begin + tid; i < end; i += threads) {
    const unsigned int key = FIRST ? map(raw[i]) : items[i].key;
    atomicAdd(&s_count[(key >> shift) & (digits - 1)], 1);
  }
  __syncthreads();
  for (int d = tid; d < digits; d += threads) counts[blockIdx.x * digits + d] = s_count[d];
}

template <bool FIRST, bool LAST, typename id_t>
__global__ void __launch_bounds__(threads)
place_digits(const int n, const id_t* __restrict__ raw, const item_t* __restrict__ items, const key_map map, const int shift, const int bits,
             const int span, const int spans, const int* __restrict__ counts, item_t* __restrict__ out, int* __restrict__ ids,
             int* __restrict__ positions) {
  typedef int quad_t __attribute__((ext_vector_type(4)));
  __shared__ int s_scan[waves];
  __shared__ quad_t s_quad[waves * max_digits / 4];
  int* const s_mem = reinterpret_cast<int*>(s_quad);
  const int digits = 1 << bits;
  const int tid = threadIdx.x;
  const int w = tid / wave::size;

  // the place of the workgroup's first item of digit `tid`: items of lower digits, and of the digit in earlier spans.  A thread adds up
  // 4 digits, the spans dealt out to slices of the threads; digits above the largest key's are left out
  const unsigned int top = static_cast<unsigned int>(map.rows) >> shift;
  const int quads = top < static_cast<unsigned int>(digits) ? static_cast<int>(top) / 4 + 1 : digits / 4;
  const int slices = threads / quads;
  const int slice = tid / quads, quad = tid % quads;
  if (slice < slices) {
    quad_t before = {0, 0, 0, 0}, total = {0, 0, 0, 0};
#pragma unroll 8
    for (int s = slice; s < spans; s += slices) {
      const quad_t c = *reinterpret_cast<const quad_t*>(counts + static_cast<std::size_t>(s) * digits + 4 * quad);
      total += c;
      before += s < static_cast<int>(blockIdx.x) ? c : quad_t{0, 0, 0, 0};
    }
    s_quad[slice * quads + quad] = before;  // [2][slices][quads]
    s_quad[threads + slice * quads + quad] = total;
  }
  __syncthreads();
  int before = 0, total = 0;
  if (tid < 4 * quads)
    for (int s = 0; s < slices; ++s) {
      before += s_mem[4 * s * quads + tid];
      total += s_mem[4 * threads + 4 * s * quads + tid];
    }
  const int base = detail::block_exclusive_sum(total, s_scan) + before;  // (its barriers end the use of s_mem)

  // the workgroup's span, a sixteenth of it (a multiple of 64 items: span is a multiple of 1 024) per wavefront
  int* const s_count = s_mem;  // [waves][digits]
  int* const mine = s_count + w * digits;
  for (int i = tid; i < waves * digits; i += threads) s_count[i] = 0;
  __syncthreads();
  const int begin = static_cast<int>(blockIdx.x) * span;
  const int size = n - begin < span ? n - begin : span;
  const int part = span / waves;
  const int wave_begin = w * part < size ? w * part : size;
  const int wave_end = wave_begin + part < size ? wave_begin + part : size;
  for (int i = wave_begin + wave::lane(); i < wave_end; i += wave::size) {
    const unsigned int key = FIRST ? map(raw[begin + i]) : items[begin + i].key;
    atomicAdd(&mine[(key >> shift) & (digits - 1)], 1);
  }
  __syncthreads();
  detail::places(s_count, digits, base);
  __syncthreads();
  for (int i = wave_begin; i < wave_end; i += wave::size) {
    const int at_item = i + wave::lane();
    const bool valid = at_item < wave_end;
    item_t it{0u, 0};
    if (valid) it = read_item<FIRST>(raw, items, map, begin + at_item);
    const int at = detail::take(mine, (it.key >> shift) & (digits - 1), bits, valid);
    if (valid) {
      if constexpr (LAST) {
        ids[at] = static_cast<int>(it.key);
        positions[at] = it.position;
      } else {
        out[at] = it;
      }
    }
  }
}

/// Enqueues the whole sort; ids / positions: n ints each.  Returns a hipError_t.
template <typename id_t>
int launch(hipStream_t stream, int n, const id_t* in, const key_map& map, int* ids, int* positions, void* workspace) {
  if (n == 0) return 0;
  const plan_t p = plan_for(n, map.rows);
  if (p.passes == 0) {
    rank<id_t><<<(n + rank_group - 1) / rank_group, threads, 0, stream>>>(n, in, map, ids, positions);
    return static_cast<int>(hipGetLastError());
  }
  char* const at = static_cast<char*>(workspace);
  const int buffers = p.passes > 2 ? 2 : p.passes - 1;
  item_t* const half[2] = {reinterpret_cast<item_t*>(at), reinterpret_cast<item_t*>(at + (buffers > 1 ? item_bytes(n) : 0))};
  int* const counts = reinterpret_cast<int*>(at + item_bytes(n) * static_cast<std::size_t>(buffers));
  const auto pass = [&](auto first_tag, auto last_tag, int index) {
    constexpr bool FIRST = decltype(first_tag)::value, LAST = decltype(last_tag)::value;
    const int shift = index * p.bits;
    const item_t* const from = FIRST ? nullptr : half[(index + 1) & 1];
    count_digits<FIRST, id_t><<<p.spans, threads, 0, stream>>>(n, in, from, map, shift, p.bits, p.span, counts);
    place_digits<FIRST, LAST, id_t><<<p.spans, threads, 0, stream>>>(n, in, from, map, shift, p.bits, p.span, p.spans, counts, half[index & 1], ids,
                                                                    positions);
  };
  for (int i = 0; i < p.passes; ++i) {
    const bool last = i == p.passes - 1;
    if (i == 0 && last) pass(std::true_type{}, std::true_type{}, i);
    else if (i == 0) pass(std::true_type{}, std::false_type{}, i);
    else if (last) pass(std::false_type{}, std::true_type{}, i);
    else pass(std::false_type{}, std::false_type{}, i);
  }
  return static_cast<int>(hipGetLastError());
}

}  // namespace group_ids
}  // namespace kernels
}  // namespace loops
