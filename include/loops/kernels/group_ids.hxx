/**
 * @file group_ids.hxx
 * @brief Groups positions by id: a stable sort of (id, position), which is the COO -> CSC conversion of a matrix with one nonzero per
 * position (row = position, column = id).  What the embedding gradient sums over and what experts' products are dispatched by.
 *
 * key(i) = id_i - first for ids in [first, first + rows) other than `drop`, `rows` otherwise (those end up behind the last group).
 * Least-significant-digit radix sort, digits of at most 10 bits, ceil(log2(rows + 1) / digits) of them:
 *
 *   n <= 8 192   ONE workgroup keeps keys and positions in LDS through all passes: one launch.
 *   beyond       two launches a pass.  COUNT: workgroup w counts the digits of its span (n / W consecutive items, W <= 256).  PLACE:
 *                every workgroup adds the counts of the spans before it by itself (W x digits words from L2; no scan launch), then each
 *                of its 16 wavefronts counts and places its own sixteenth of the span.
 *
 * A wavefront ranks 64 items at a time without atomics: one ballot per digit bit leaves each lane the mask of the lanes with its digit;
 * the rank is the number of mask bits below the lane and the last of them advances the wavefront's counter in LDS.  Items are taken in
 * order, so equal ids keep the order of their positions and the result is the same in every run.
 */
#pragma once

#include <atomic>
#include <cstddef>
#include <cstdint>

#include <hip/hip_runtime.h>

#include <loops/util/wave.hxx>

namespace loops {
namespace kernels {
namespace group_ids {

constexpr int threads = 1024;
constexpr int waves = threads / wave::size;
constexpr int max_digit_bits = 10;
constexpr int max_digits = 1 << max_digit_bits;
constexpr int block_items = 8192;  ///< what one workgroup sorts in LDS
constexpr int max_spans = 256;

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
  int passes;
  int bits;   ///< per digit
  int spans;  ///< workgroups of a COUNT / PLACE launch (1: everything in one workgroup)
  int span;   ///< items per workgroup
};

/// Bits are shared out evenly: 18 bits are two digits of 9.  A span is at least 4 096 items (four rounds per wavefront) and there
/// are at most 256, so that the counts a PLACE workgroup adds up stay within 1 MB.
inline plan_t plan_for(int n, int rows) {
  int bits = 1;
  while (bits < 31 && (static_cast<unsigned int>(rows) >> bits) != 0u) ++bits;
  plan_t p;
  p.passes = (bits + max_digit_bits - 1) / max_digit_bits;
  p.bits = (bits + p.passes - 1) / p.passes;
  p.spans = 1;
  p.span = n;
  if (n > block_items) {
    const int want = (n + 4095) / 4096;
    const int w = want < max_spans ? want : max_spans;
    const long long per = (static_cast<long long>(n) + w - 1) / w;
    p.span = static_cast<int>((per + threads - 1) / threads * threads);
    p.spans = static_cast<int>((static_cast<long long>(n) + p.span - 1) / p.span);
  }
  return p;
}

inline std::size_t workspace_bytes(int n, int rows) {
  const plan_t p = plan_for(n, rows);
  if (p.spans == 1) return 0;
  const std::size_t items = (static_cast<std::size_t>(n) * sizeof(item_t) + 255) & ~static_cast<std::size_t>(255);
  return items * static_cast<std::size_t>(p.passes > 2 ? 2 : p.passes - 1) + static_cast<std::size_t>(p.spans) * (static_cast<std::size_t>(1) << p.bits) * sizeof(int);
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

/// n <= IPT * 1 024 items, all passes in one workgroup.  Item j of wavefront w, lane l is w * 64 * IPT + j * 64 + l.
template <int IPT, typename id_t>
__global__ void __launch_bounds__(threads)
sort_block(const int n, const id_t* __restrict__ in, const key_map map, const int passes, const int bits, int* __restrict__ ids,
           int* __restrict__ positions) {
  extern __shared__ int s_mem[];
  const int digits = 1 << bits;
  int* const s_scan = s_mem;                // [16]
  int* const s_count = s_mem + waves;       // [waves][digits]
  unsigned int* const s_key = reinterpret_cast<unsigned int*>(s_count + waves * digits);  // [n]
  int* const s_position = reinterpret_cast<int*>(s_key + IPT * threads);                  // [n]
  const int tid = threadIdx.x;
  const int w = tid / wave::size;
  const int first = w * wave::size * IPT + wave::lane();
  int* const mine = s_count + w * digits;

  unsigned int key[IPT];
  int position[IPT];
#pragma unroll
  for (int j = 0; j < IPT; ++j) {
    const int i = first + j * wave::size;
    position[j] = i;
    key[j] = i < n ? map(in[i]) : 0u;
  }
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = pass * bits;
    for (int i = tid; i < waves * digits; i += threads) s_count[i] = 0;
    __syncthreads();
    int rank[IPT];  // among the wavefront's items of the digit
#pragma unroll
    for (int j = 0; j < IPT; ++j)
      rank[j] = detail::take(mine, (key[j] >> shift) & (digits - 1), bits, first + j * wave::size < n);
    __syncthreads();
    int total = 0;
    if (tid < digits)
      for (int v = 0; v < waves; ++v) total += s_count[v * digits + tid];
    const int base = detail::block_exclusive_sum(total, s_scan);
    detail::places(s_count, digits, base);
    __syncthreads();
    const bool last = pass == passes - 1;
#pragma unroll
    for (int j = 0; j < IPT; ++j) {
      if (first + j * wave::size < n) {
        const int at = mine[(key[j] >> shift) & (digits - 1)] + rank[j];
        if (last) {
          ids[at] = static_cast<int>(key[j]);
          positions[at] = position[j];
        } else {
          s_key[at] = key[j];
          s_position[at] = position[j];
        }
      }
    }
    if (!last) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < IPT; ++j) {
        const int i = first + j * wave::size;
        if (i < n) {
          key[j] = s_key[i];
          position[j] = s_position[i];
        }
      }
      __syncthreads();
    }
  }
}

/// sort_block's launch.  Its LDS is up to 128 KB (10-bit digits, 8 192 items): beyond 64 KB a kernel is opted in once per device.
template <int IPT, typename id_t>
void launch_sort_block(hipStream_t stream, int n, const id_t* in, const key_map& map, const plan_t& p, int* ids, int* positions) {
  static std::atomic<unsigned long long> opted{0ull};
  const std::size_t items = p.passes > 1 ? 2u * IPT * threads : 0u;
  const std::size_t lds = sizeof(int) * (waves + static_cast<std::size_t>(waves) * (static_cast<std::size_t>(1) << p.bits) + items);
  if (lds > 64 * 1024) {
    int device = 0;
    const bool known = hipGetDevice(&device) == hipSuccess && device >= 0 && device < 64;
    if (!known || !((opted.load() >> device) & 1ull)) {
      (void)hipFuncSetAttribute(reinterpret_cast<const void*>(&sort_block<IPT, id_t>), hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
      if (known) opted.fetch_or(1ull << device);
    }
  }
  sort_block<IPT, id_t><<<1, threads, lds, stream>>>(n, in, map, p.passes, p.bits, ids, positions);
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
  __shared__ int s_scan[waves];
  __shared__ int s_count[waves * max_digits];
  const int digits = 1 << bits;
  const int tid = threadIdx.x;
  const int w = tid / wave::size;
  int* const mine = s_count + w * digits;
  for (int i = tid; i < waves * digits; i += threads) s_count[i] = 0;
  __syncthreads();

  // the workgroup's span, a sixteenth of it (a multiple of 64 items: span is a multiple of 1 024) per wavefront
  const int begin = blockIdx.x * span;
  const int size = n - begin < span ? n - begin : span;
  const int part = span / waves;
  const int wave_begin = w * part < size ? w * part : size;
  const int wave_end = wave_begin + part < size ? wave_begin + part : size;
  for (int i = wave_begin + wave::lane(); i < wave_end; i += wave::size) {
    const unsigned int key = FIRST ? map(raw[begin + i]) : items[begin + i].key;
    atomicAdd(&mine[(key >> shift) & (digits - 1)], 1);
  }
  int before = 0, total = 0;  // items of digit `tid` in the spans before this one / in all
  if (tid < digits) {
#pragma unroll 8
    for (int s = 0; s < spans; ++s) {
      const int c = counts[s * digits + tid];
      total += c;
      before += s < static_cast<int>(blockIdx.x) ? c : 0;
    }
  }
  const int base = detail::block_exclusive_sum(total, s_scan) + before;  // (its barriers also order the counts above)
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
  if (p.spans == 1) {
    if (n <= threads) launch_sort_block<1, id_t>(stream, n, in, map, p, ids, positions);
    else if (n <= 4 * threads) launch_sort_block<4, id_t>(stream, n, in, map, p, ids, positions);
    else launch_sort_block<8, id_t>(stream, n, in, map, p, ids, positions);
    return static_cast<int>(hipGetLastError());
  }
  const std::size_t stride = (static_cast<std::size_t>(n) * sizeof(item_t) + 255) & ~static_cast<std::size_t>(255);
  char* const at = static_cast<char*>(workspace);
  const int buffers = p.passes > 2 ? 2 : p.passes - 1;
  item_t* const half[2] = {reinterpret_cast<item_t*>(at), reinterpret_cast<item_t*>(at + (buffers > 1 ? stride : 0))};
  int* const counts = reinterpret_cast<int*>(at + stride * static_cast<std::size_t>(buffers));
  for (int pass = 0; pass < p.passes; ++pass) {
    const int shift = pass * p.bits;
    const item_t* const from = half[(pass + 1) & 1];
    item_t* const to = half[pass & 1];
    const bool last = pass == p.passes - 1;
    if (pass == 0) {
      count_digits<true, id_t><<<p.spans, threads, 0, stream>>>(n, in, nullptr, map, shift, p.bits, p.span, counts);
      if (last)
        place_digits<true, true, id_t><<<p.spans, threads, 0, stream>>>(n, in, nullptr, map, shift, p.bits, p.span, p.spans, counts, nullptr, ids, positions);
      else
        place_digits<true, false, id_t><<<p.spans, threads, 0, stream>>>(n, in, nullptr, map, shift, p.bits, p.span, p.spans, counts, to, nullptr, nullptr);
    } else {
      count_digits<false, id_t><<<p.spans, threads, 0, stream>>>(n, nullptr, from, map, shift, p.bits, p.span, counts);
      if (last)
        place_digits<false, true, id_t><<<p.spans, threads, 0, stream>>>(n, nullptr, from, map, shift, p.bits, p.span, p.spans, counts, nullptr, ids, positions);
      else
        place_digits<false, false, id_t><<<p.spans, threads, 0, stream>>>(n, nullptr, from, map, shift, p.bits, p.span, p.spans, counts, to, nullptr, nullptr);
    }
  }
  return static_cast<int>(hipGetLastError());
}

}  // namespace group_ids
}  // namespace kernels
}  // namespace loops
