/**
 * @file embedding.hxx
 * @brief Embedding of tokens and its gradient: the product of the token matrix S (tokens x rows of the table, one 1 per token) with the
 * table, and of its transpose with the gradient of the output.
 *
 *   lookup     out[t, :]   = scale * table[id_t - first, :]      (zeros for ids outside [first, first + rows))
 *   gradient   grad[v, :]  = scale * sum over the tokens of row v of out_grad[t, :]  (+ grad[v, :])
 *
 * Both only move bytes: HBM bounds them.  Sums are held in float and rounded once, when the row is stored.
 */
#pragma once

#include <climits>
#include <cstddef>
#include <cstdint>
#include <type_traits>

#include <hip/hip_runtime.h>

#include <loops/kernels/group_ids.hxx>
#include <loops/util/elements.hxx>
#include <loops/util/wave.hxx>

namespace loops {
namespace kernels {
namespace embedding {

/// Threads that one dimension of a grid holds.
constexpr unsigned long long max_launch_threads = (1ull << 32) - 1;
/// Columns of one launch: the kernels' column numbers and grids stay within 32 bits (the gradient's of 16 threads per column the closest).
constexpr int max_columns = 1 << 27;

/// f(at, cols) for the column ranges [at, at + cols) of a matrix, until one returns an error: all columns at once up to max_columns.
template <typename F>
int by_columns(int dim, F&& f) {
  for (int at = 0;;) {
    const int cols = dim - at < max_columns ? dim - at : max_columns;
    const int err = f(at, cols);
    if (err || dim - at == cols) return err;
    at += cols;
  }
}

// ---- lookup -------------------------------------------------------------------------------------------------------------------
constexpr int lookup_threads = 256;

/**
 * A row is cut into `packets` = ceil(dim / V) packets of V values, the last one shifted back to end with the row (its overlap is
 * written twice, with the same values): any width and alignment moves in 16-byte accesses.  Packets of all rows are numbered through
 * and each thread takes U of them, a workgroup's width apart: consecutive lanes touch consecutive packets whatever the width.
 * HBM bounds it: 65 536 tokens of a 131 072 x 2 048 float table in 125 us where ids fall off as in text (20 079 different rows: 5.6 TB/s of what
 * has to move), 162 where they are uniform (51 665: 5.9); 16 tokens take 2.4 us, a launch.
 */
template <int V, int U, bool STREAM, typename type_t, typename id_t>
__global__ void __launch_bounds__(lookup_threads)
lookup(const type_t* __restrict__ table, const std::size_t table_pitch, const id_t* __restrict__ ids, const int tokens, const int packets,
       const int dim, const group_ids::key_map map, const float scale, type_t* __restrict__ out, const std::size_t out_pitch) {
  const unsigned long long begin = static_cast<unsigned long long>(blockIdx.x) * (lookup_threads * U);
  const unsigned int width = static_cast<unsigned int>(packets);
  unsigned int token0 = 0, offset = 0;  // of the workgroup's first packet
  if (begin >> 32) {
    token0 = static_cast<unsigned int>(begin / width);
    offset = static_cast<unsigned int>(begin % width);
  } else {
    token0 = static_cast<unsigned int>(begin) / width;
    offset = static_cast<unsigned int>(begin) % width;
  }
  unsigned int token[U], column[U];
  unsigned int row[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const unsigned int i = offset + u * lookup_threads + threadIdx.x;
    const unsigned int t = i / width;
    const unsigned int c = (i - t * width) * V;
    token[u] = token0 + t;
    column[u] = c + V <= static_cast<unsigned int>(dim) ? c : static_cast<unsigned int>(dim - V);
    row[u] = token[u] < static_cast<unsigned int>(tokens) ? map(ids[token[u]]) : static_cast<unsigned int>(map.rows);
  }
  elements::packet_t<type_t, V> packet[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    packet[u] = elements::packet_t<type_t, V>{};
    if (row[u] < static_cast<unsigned int>(map.rows)) packet[u] = elements::load<V>(table + row[u] * table_pitch + column[u]);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (token[u] < static_cast<unsigned int>(tokens)) {
      const bool inside = row[u] < static_cast<unsigned int>(map.rows);
      float v[V];
#pragma unroll
      for (int k = 0; k < V; ++k) v[k] = inside ? static_cast<float>(packet[u][k]) * scale : 0.0f;
      elements::store<V, STREAM>(out + token[u] * out_pitch + column[u], v);
    }
  }
}

template <typename type_t, typename id_t>
int launch_lookup(hipStream_t stream, const type_t* table, std::size_t table_pitch, const id_t* ids, int tokens, int dim,
                  const group_ids::key_map& map, float scale, type_t* out, std::size_t out_pitch) {
  if (tokens == 0 || dim == 0) return 0;
  constexpr int V = elements::per_access<type_t>;
  // columns [at, at + cols) of all tokens, in as few launches as hold them (one but for some 2^32 packets)
  const auto run = [&](auto v_tag, auto u_tag, auto stream_tag, int at, int cols) {
    constexpr int W = decltype(v_tag)::value, U = decltype(u_tag)::value;
    const int packets = (cols + W - 1) / W;
    const long long most = static_cast<long long>(max_launch_threads / lookup_threads) * (lookup_threads * U) / packets;
    for (long long t = 0; t < tokens; t += most) {
      const int count = static_cast<int>(tokens - t < most ? tokens - t : most);
      const unsigned long long all = static_cast<unsigned long long>(count) * packets;
      const unsigned int grid = static_cast<unsigned int>((all + lookup_threads * U - 1) / (lookup_threads * U));
      lookup<W, U, decltype(stream_tag)::value, type_t, id_t><<<grid, lookup_threads, 0, stream>>>(
          table + at, table_pitch, ids + t, count, packets, cols, map, scale, out + static_cast<std::size_t>(t) * out_pitch + at, out_pitch);
      if (const hipError_t err = hipGetLastError()) return static_cast<int>(err);
    }
    return 0;
  };
  using one = std::integral_constant<int, 1>;
  using width = std::integral_constant<int, V>;
  // Four packets per thread where that still fills the chip (bf16, dim 4 096: 512 tokens 3.4 us with one, 4.2 with four; 2 048: 6.6, 6.1;
  // 16 384: 48.5, 41.0).  Stores of whole lines go past the caches (65 536 x 2 048 float, uniform ids: 160 us, 198 through them); others are left to the
  // L2 to gather.
  const bool whole_lines = (reinterpret_cast<std::uintptr_t>(out) | (out_pitch * sizeof(type_t)) | (dim * sizeof(type_t))) % 128 == 0;
  const bool many = static_cast<unsigned long long>(tokens) * dim >= 512ull * lookup_threads * 4 * V;
  return by_columns(dim, [&](int at, int cols) {
    if (cols < V) return run(one{}, one{}, std::false_type{}, at, cols);
    if (!many) return run(width{}, one{}, std::false_type{}, at, cols);
    return whole_lines ? run(width{}, std::integral_constant<int, 4>{}, std::true_type{}, at, cols)
                       : run(width{}, std::integral_constant<int, 4>{}, std::false_type{}, at, cols);
  });
}

// ---- gradient -----------------------------------------------------------------------------------------------------------------
constexpr int gradient_threads = 256;
constexpr int gradient_waves = gradient_threads / wave::size;

/// Columns per lane: one 16-byte access of the wider of the two types, so that every store of a wavefront covers whole lines.
template <typename type_t, typename out_t>
constexpr int lane_width = elements::per_access<type_t> < elements::per_access<out_t> ? elements::per_access<type_t> : elements::per_access<out_t>;

struct gradient_plan {
  int slabs;  ///< column slabs
  int items;  ///< tokens per tile
  int tiles;
};

/// Equal tiles of the tokens sorted by row, one wavefront per (tile, slab of columns): a row of a hundred thousand tokens and a hundred
/// thousand rows of one are the same work per wavefront.  16 384 wavefronts are two for every place on the chip.
inline gradient_plan gradient_plan_for(int width, int tokens, int dim) {
  gradient_plan p;
  p.slabs = (dim + wave::size * width - 1) / (wave::size * width);
  long long items = (static_cast<long long>(tokens) * p.slabs + 16383) / 16384;
  items = items < 16 ? 16 : items > INT_MAX ? INT_MAX : items;
  p.items = static_cast<int>(items);
  p.tiles = static_cast<int>((tokens + items - 1) / items);
  return p;
}

/// What a tile leaves for the join: the row it finished that an earlier tile began, the row it began or continued and did not finish
/// (-1: none).
struct tile_record {
  int head_row;
  int tail_row;
};

/// A rule for calls that the host makes one by one: one launch instead of two, and no workspace, save it 4 us.  With the grouping before it a call
/// takes 15.3 us up to 512 tokens whatever the width (64, 1 024, 8 192 columns, bf16 into float and float; 8 192: 16.8 at 512), 18.9 at 640 (21.0) and
/// 20.0 at 768 (22.3), in two launches 19.8 at all of them.  Replayed from a graph, where the host's time is gone, the one launch is shorter up to 256
/// tokens (x 1 024: 128 6.2 us, 7.9 with the join; 256 7.3, 8.1; 384 11.4, 8.2; 512 12.2, 8.1; 640 16.1, 8.3); the rule is the same there, as the two
/// forms add in different orders and equal inputs give equal bits.
constexpr int small_tokens = 640;  ///< most tokens of add_small

/// Workspace: records[tiles], heads[tiles][dim], tails[tiles][dim] (float).
inline std::size_t gradient_records_bytes(int tiles) { return (static_cast<std::size_t>(tiles) * sizeof(tile_record) + 255) & ~static_cast<std::size_t>(255); }
template <typename type_t, typename out_t>
std::size_t gradient_workspace_bytes(int tokens, int rows, int dim, bool add) {
  if (dim == 0 || rows == 0 || (add && tokens <= small_tokens)) return 0;
  std::size_t most = 0;  // column ranges follow each other in the same memory
  by_columns(dim, [&](int, int cols) {
    const gradient_plan p = gradient_plan_for(lane_width<type_t, out_t>, tokens, cols);
    const std::size_t bytes = gradient_records_bytes(p.tiles) + 2 * static_cast<std::size_t>(p.tiles) * cols * sizeof(float);
    most = bytes > most ? bytes : most;
    return 0;
  });
  return most;
}

/// Ids and positions that group_ids did not write are not followed out of the arrays, whatever they are: positions are bounded, ids count
/// up to the first that is no row (`leading` of the lanes that hold one).
__device__ __forceinline__ bool is_row(int key, int rows) { return static_cast<unsigned int>(key) < static_cast<unsigned int>(rows); }
__device__ __forceinline__ int leading(unsigned long long lanes) { return lanes == ~0ull ? wave::size : __builtin_ctzll(~lanes); }
__device__ __forceinline__ int bounded(int position, int tokens) {
  return static_cast<unsigned int>(position) < static_cast<unsigned int>(tokens) ? position : 0;
}

/// The number of keys below `row`.  All lanes search together, 64 probes a step.
__device__ __forceinline__ int keys_below(const int* __restrict__ keys, int tokens, int row) {
  int lo = 0, hi = tokens;  // answer in [lo, hi]
  while (hi > lo) {
    const int step = (hi - lo + wave::size - 1) / wave::size;
    const long long probe = static_cast<long long>(lo) + static_cast<long long>(wave::lane()) * step;
    const int n = leading(__ballot(probe < hi && keys[probe < hi ? probe : lo] < row));
    if (n == 0) return lo;
    const long long next_hi = static_cast<long long>(lo) + static_cast<long long>(n) * step;
    lo = lo + (n - 1) * step + 1;
    hi = next_hi < hi ? static_cast<int>(next_hi) : hi;
  }
  return lo;
}

/// A row of fewer tokens than this belongs to the tile of its first token; longer ones are cut at the tiles' ends and joined.
constexpr int whole_row = wave::size;

/// The columns of a lane in slab `part`; the last packet of a row is shifted back to end with it and keeps its own columns only.
template <int V>
struct lane_columns {
  int at;
  int skip;  ///< elements of the packet before the lane's own (V: none is the lane's)
  bool whole;
  __device__ __forceinline__ lane_columns(int part, int dim) {
    const int own = (part * wave::size + wave::lane()) * V;
    whole = own + V <= dim;
    const bool active = own < dim;
    at = whole ? own : active ? dim - V : 0;
    skip = active ? own - at : V;
  }
  template <bool STREAM = false, typename T>
  __device__ __forceinline__ void store(T* __restrict__ row, const float (&v)[V]) const {
    if (whole) {
      elements::store<V, STREAM>(row + at, v);
    } else {
#pragma unroll
      for (int k = 0; k < V; ++k)
        if (k >= skip) row[at + k] = static_cast<T>(v[k]);
    }
  }
};

/// How many of the 64 tokens from `at` on (before it, for before = true) have this key.
template <bool BEFORE>
__device__ __forceinline__ int same_key(const int* __restrict__ keys, int tokens, int at, int key) {
  const int j = BEFORE ? at - 1 - wave::lane() : at + wave::lane();
  return __popcll(__ballot(j >= 0 && j < tokens && keys[j < 0 ? 0 : j < tokens ? j : tokens - 1] == key));
}

/// How the rows without a token are dealt out to clearing workgroups: `rows` of them together, or a row in `parts`.
struct clear_plan {
  int rows;
  int parts;
  long long groups;
};

constexpr int clear_rows = gradient_threads;  ///< most rows per clearing workgroup

/// Stores that go past the caches (`stream`): pieces of 8 KB, so that what the workgroups write at one time is close to one stretch of memory
/// (131 072 rows of 8 KB, the whole pass: 186 us; pieces of 4 KB, half of whose time is the search for their rows, 292, of 16 KB 211, of 128
/// KB 219).  Stores that the L2 gathers: 32 KB (50 021 rows of 4 004 bytes: 63 us; 8 KB 68, 16 and 64 KB 64).  More where the grid would
/// not hold them.
inline clear_plan clear_plan_for(int rows, std::size_t row_bytes, bool stream) {
  clear_plan p;
  for (std::size_t piece = stream ? 8192 : 32768;; piece *= 2) {
    p.rows = row_bytes >= piece ? 1 : piece / row_bytes > clear_rows ? clear_rows : static_cast<int>(piece / row_bytes);
    p.parts = static_cast<int>((row_bytes * p.rows + piece - 1) / piece);
    p.groups = (static_cast<long long>(rows) + p.rows - 1) / p.rows * p.parts;
    if (p.groups <= 3 << 22 || p.rows == clear_rows) return p;
  }
}

/// Zeros into those of the rows of clearing workgroup `group` that have no token.
template <bool STREAM, typename out_t>
__device__ __forceinline__ void clear_empty(const int* __restrict__ keys, int tokens, int rows, const clear_plan& plan, unsigned int group, int dim,
                                            out_t* __restrict__ grad, std::size_t grad_pitch) {
  __shared__ int s_range[2];
  __shared__ int s_has[clear_rows];
  const int tid = threadIdx.x;
  const unsigned int place = group / plan.parts, part = group - place * plan.parts;
  const int begin = static_cast<int>(place) * plan.rows;
  const int count = rows - begin < plan.rows ? rows - begin : plan.rows, end = begin + count;
  s_has[tid] = 0;
  const int w = __builtin_amdgcn_readfirstlane(tid / wave::size);
  if (w < 2) {
    const int at = keys_below(keys, tokens, w == 0 ? begin : end);
    if (wave::lane() == 0) s_range[w] = at;
  }
  __syncthreads();
  const int lo = s_range[0], hi = s_range[1];
  if (count == 1) {
    if (hi > lo) return;
  } else if (hi - lo <= 4 * gradient_threads) {
    for (int j = lo + tid; j < hi; j += gradient_threads) {
      const unsigned int row = static_cast<unsigned int>(keys[j] - begin);
      if (row < static_cast<unsigned int>(count)) s_has[row] = 1;
    }
  } else if (tid < count) {  // rows of many tokens: each is searched for
    int l = lo, h = hi;
    while (l < h) {
      const int m = l + (h - l) / 2;
      if (keys[m] < begin + tid) l = m + 1;
      else h = m;
    }
    s_has[tid] = l < hi && keys[l] == begin + tid;
  }
  __syncthreads();
  const auto fill = [&](auto v_tag) {
    constexpr int V = decltype(v_tag)::value;
    const unsigned int packets = (dim + V - 1) / V, all = packets * count;  // (parts > 1: one row)
    const unsigned int per_part = (packets + plan.parts - 1) / plan.parts;
    const unsigned int first = plan.parts > 1 ? part * per_part : 0, last = plan.parts > 1 && first + per_part < all ? first + per_part : all;
    const float zero[V] = {};
    for (unsigned int i = first + tid; i < last; i += gradient_threads) {
      const unsigned int row = i / packets;
      const int own = static_cast<int>(i - row * packets) * V;
      if (!s_has[row]) elements::store<V, STREAM>(grad + static_cast<std::size_t>(begin + row) * grad_pitch + (own + V <= dim ? own : dim - V), zero);
    }
  };
  if (dim >= elements::per_access<out_t>) fill(std::integral_constant<int, elements::per_access<out_t>>{});
  else fill(std::integral_constant<int, 1>{});
}

/**
 * One wavefront per (tile, slab); 64 tokens' keys and positions are loaded at a time, one per lane, and become scalars as the wavefront
 * walks over them with U gradient rows in flight.  ADD: rows with tokens are added to; what a row held is read together with the gradient
 * row of its last token, so that the two latencies are one.  Otherwise rows with tokens are written, and the workgroups behind the tiles'
 * write zeros into the others, in the order of memory: rows cleared from within the tiles, as they came in the list, left the chip at 5.2
 * TB/s (8 192 tokens, 131 072 rows of 8 KB: 203 us, now 172, 6.6 TB/s).
 * 8 wavefronts per SIMD are asked for: scalar registers would allow 7 otherwise (131 072 tokens x 4 096 bf16 into float, whole pass: 670
 * us, 632 with 8: 5.1 TB/s of reads and writes together, where a copy of 4 GiB reaches 4.7).
 * ADD at the same size, 32 600 different rows: 471 us, 4.5 TB/s, the copy's rate; 8 rows in flight (475), 8 wavefronts asked for (473) and stores past
 * the caches (470 to 475) leave it there.
 */
template <bool ADD, int V, int U, bool STREAM, typename type_t, typename out_t>
__global__ void __launch_bounds__(gradient_threads, ADD ? 1 : 8)
gradient(const int* __restrict__ keys, const int* __restrict__ positions, const int tokens, const int rows, const type_t* __restrict__ from,
         const std::size_t from_pitch, const int dim, const float scale, out_t* __restrict__ grad, const std::size_t grad_pitch, const int tiles,
         const int items, const int slabs, const unsigned int tile_groups, const clear_plan clear, tile_record* __restrict__ records,
         float* __restrict__ heads, float* __restrict__ tails) {
  if constexpr (!ADD) {
    if (blockIdx.x >= tile_groups) {
      clear_empty<STREAM>(keys, tokens, rows, clear, blockIdx.x - tile_groups, dim, grad, grad_pitch);
      return;
    }
  }
  const int unit = __builtin_amdgcn_readfirstlane(static_cast<int>(blockIdx.x) * gradient_waves + static_cast<int>(threadIdx.x) / wave::size);
  const int tile = unit / slabs;
  if (tile >= tiles) return;
  const int part = unit - tile * slabs;
  const lane_columns<V> cols(part, dim);
  const long long d0 = static_cast<long long>(tile) * items;
  int y = static_cast<int>(d0);
  const int end = d0 + items < tokens ? static_cast<int>(d0 + items) : tokens;
  int row = keys[y];
  bool open = false;  // the row was begun by an earlier tile, and is cut here
  if (y > 0 && is_row(row, rows) && keys[y - 1] == row) {
    const int behind = same_key<false>(keys, tokens, y, row);
    open = same_key<true>(keys, tokens, y, row) + behind >= whole_row;
    if (!open) y += behind;
  }
  int begun = y;  // the row's first token here
  int head_row = -1;
  float acc[V];
#pragma unroll
  for (int k = 0; k < V; ++k) acc[k] = 0.0f;

  const auto consume = [&](int key, int position, unsigned long long last, int count) {  // tokens y .. y + count; last: bits of the rows' ends
    for (int i = 0; i < count; i += U) {
      elements::packet_t<type_t, V> packet[U];
      elements::packet_t<out_t, V> old[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int at = i + u < count ? i + u : count - 1;
        packet[u] = elements::load<V>(from + static_cast<std::size_t>(__builtin_amdgcn_readlane(position, at)) * from_pitch + cols.at);
        if (ADD && ((last >> at) & 1ull)) old[u] = elements::load<V>(grad + static_cast<std::size_t>(__builtin_amdgcn_readlane(key, at)) * grad_pitch + cols.at);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (i + u < count) {
#pragma unroll
          for (int c = 0; c < V; ++c) acc[c] += static_cast<float>(packet[u][c]);
          if ((last >> (i + u)) & 1ull) {
            const int k = __builtin_amdgcn_readlane(key, i + u);
            if (open) {
              head_row = k;
              cols.store(heads + static_cast<std::size_t>(tile) * dim, acc);
              open = false;
            } else {
              float v[V];
#pragma unroll
              for (int c = 0; c < V; ++c) v[c] = ADD ? __builtin_fmaf(scale, acc[c], static_cast<float>(old[u][c])) : scale * acc[c];
              cols.template store<STREAM>(grad + static_cast<std::size_t>(k) * grad_pitch, v);
            }
#pragma unroll
            for (int c = 0; c < V; ++c) acc[c] = 0.0f;
            begun = y + i + u + 1;
          }
        }
      }
    }
    y += count;
  };

  while (y < end) {
    const int j = y + wave::lane();
    int key = rows, next = rows, position = 0;
    if (j < tokens) {
      key = keys[j];
      position = bounded(positions[j], tokens);
      if (j + 1 < tokens) next = keys[j + 1];
    }
    const int count = leading(__ballot(is_row(key, rows) && j < end));
    if (count == 0) break;
    const unsigned long long last = __ballot(key != next);
    row = __builtin_amdgcn_readlane(key, count - 1);
    consume(key, position, last, count);
    if (count < wave::size) break;
  }
  bool unfinished = y > begun;
  if (unfinished && !open) {
    const int behind = same_key<false>(keys, tokens, y, row);  // (at least one: the row's last token was not the tile's)
    if (y - begun + behind < whole_row) {
      const int j = y + wave::lane();
      consume(row, j < tokens ? bounded(positions[j], tokens) : 0, 1ull << (behind - 1), behind);
      unfinished = false;
    }
  }
  if (unfinished) cols.store(tails + static_cast<std::size_t>(tile) * dim, acc);
  if (part == 0 && wave::lane() == 0) records[tile] = tile_record{head_row, unfinished ? row : -1};
}

constexpr int small_threads = 1024;
constexpr int small_waves = small_threads / wave::size;
static_assert(small_tokens <= small_waves * wave::size, "a token per lane");

/**
 * gradient<ADD> for few tokens, in one launch: a workgroup adds all tokens of 64 columns, a sixteenth of them per wavefront, and rows
 * that several wavefronts hold are joined in LDS.  One column per lane: a row of the gradient is spread over as many CUs as there are
 * slabs (1 024 columns: 16), which few tokens leave idle otherwise.
 */
template <int U, typename type_t, typename out_t>
__global__ void __launch_bounds__(small_threads)
add_small(const int* __restrict__ keys, const int* __restrict__ positions, const int tokens, const int rows,
                   const type_t* __restrict__ from, const std::size_t from_pitch, const int dim, const float scale, out_t* __restrict__ grad,
                   const std::size_t grad_pitch) {
  __shared__ float s_tail[small_waves][wave::size];
  __shared__ int s_tail_row[small_waves];
  const int w = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / wave::size);
  const int lane = wave::lane();
  const int column = static_cast<int>(blockIdx.x) * wave::size + lane;
  const bool active = column < dim;
  const int at = active ? column : 0;
  const int items = (tokens + small_waves - 1) / small_waves;  // at most 64: a token per lane
  const int begin = w * items < tokens ? w * items : tokens;
  const int end = begin + items < tokens ? begin + items : tokens;
  const int j = begin + lane;
  int key = rows, next = rows, position = 0;
  if (j < end) {
    key = keys[j];
    position = bounded(positions[j], tokens);
    if (j + 1 < tokens) next = keys[j + 1];
  }
  const int count = leading(__ballot(is_row(key, rows)));
  const unsigned long long last = __ballot(key != next);
  bool open = count > 0 && begin > 0 && keys[begin - 1] == __builtin_amdgcn_readfirstlane(key);
  int head_row = -1;
  float acc = 0.0f, head = 0.0f, head_old = 0.0f;
  for (int i = 0; i < count; i += U) {
    type_t value[U];
    out_t old[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int t = i + u < count ? i + u : count - 1;
      value[u] = from[static_cast<std::size_t>(__builtin_amdgcn_readlane(position, t)) * from_pitch + at];
      old[u] = grad[static_cast<std::size_t>(__builtin_amdgcn_readlane(key, t)) * grad_pitch + at];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u < count) {
        acc += static_cast<float>(value[u]);
        if ((last >> (i + u)) & 1ull) {
          const int row = __builtin_amdgcn_readlane(key, i + u);
          if (open) {
            head_row = row;
            head = acc;
            head_old = static_cast<float>(old[u]);
            open = false;
          } else if (active) {
            grad[static_cast<std::size_t>(row) * grad_pitch + at] = static_cast<out_t>(__builtin_fmaf(scale, acc, static_cast<float>(old[u])));
          }
          acc = 0.0f;
        }
      }
    }
  }
  const bool unfinished = count > 0 && !((last >> (count - 1)) & 1ull);
  s_tail[w][lane] = acc;
  if (lane == 0) s_tail_row[w] = unfinished ? __builtin_amdgcn_readlane(key, count > 0 ? count - 1 : 0) : -1;
  __syncthreads();
  if (head_row >= 0 && active) {
    int first = w;
    while (first > 0 && s_tail_row[first - 1] == head_row) --first;
    float sum = 0.0f;
    for (int i = first; i < w; ++i) sum += s_tail[i][lane];
    grad[static_cast<std::size_t>(head_row) * grad_pitch + at] = static_cast<out_t>(__builtin_fmaf(scale, sum + head, head_old));
  }
}

constexpr int join_threads = 512;
constexpr int join_waves = join_threads / wave::size;

/**
 * The rows that more than one tile holds: sum of the tails of the tiles before, in a fixed order, and the finishing tile's head.
 * A workgroup covers 128 columns and every gridDim.y-th tile; its wavefronts share a row's tails out.  A long row's tails are read by as many
 * CUs as it has groups of columns, which bounds it (a row of 10 000 of 20 011 tokens leaves 590 tails of 1 001 columns: 16 us at 256
 * columns per workgroup, 13 at 128, 11 at 64, where the many short joins of 131 072 x 4 096 take 4 us more).
 */
template <bool ADD, typename out_t>
__global__ void __launch_bounds__(join_threads)
join(const tile_record* __restrict__ records, const float* __restrict__ heads, const float* __restrict__ tails, const int tiles, const int dim,
     const float scale, out_t* __restrict__ grad, const std::size_t grad_pitch) {
  constexpr int C = 2;  // columns per lane
  constexpr int U = 8;
  __shared__ float s_sum[join_waves][C][wave::size];
  const int w = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / wave::size);
  const int lane = wave::lane();
  const int own = (static_cast<int>(blockIdx.x) * wave::size + lane) * C;
  const int mine = own < dim ? (dim - own < C ? dim - own : C) : 0;
  const auto read = [&](const float* __restrict__ from, int tile, float (&v)[C]) {
    const float* const at = from + static_cast<std::size_t>(tile) * dim + own;
    if (mine == C) {
      const auto p = elements::load<C>(at);
#pragma unroll
      for (int c = 0; c < C; ++c) v[c] = p[c];
    } else {
#pragma unroll
      for (int c = 0; c < C; ++c) v[c] = c < mine ? at[c] : 0.0f;
    }
  };
  const int stride = static_cast<int>(gridDim.y);
  for (int t0 = static_cast<int>(blockIdx.y); t0 < tiles; t0 += stride * wave::size) {
    const long long t = static_cast<long long>(t0) + static_cast<long long>(lane) * stride;
    const int head = t < tiles ? records[t].head_row : -1;
    unsigned long long todo = __ballot(head >= 0);
    while (todo) {
      const int at = __builtin_ctzll(todo);
      todo &= todo - 1;
      const int tile = t0 + at * stride;
      const int row = __builtin_amdgcn_readlane(head, at);
      int run = 0;  // tiles before this one that hold a part of the row
      for (;;) {
        const int b = tile - 1 - run - lane;
        const unsigned long long part = __ballot(b >= 0 && records[b < 0 ? 0 : b].tail_row == row);
        const int n = part == ~0ull ? wave::size : __builtin_ctzll(~part);
        run += n;
        if (n < wave::size) break;
      }
      float sum[C] = {};
      for (int b = tile - run + w; b < tile; b += join_waves * U) {
        float v[U][C];
#pragma unroll
        for (int u = 0; u < U; ++u) read(tails, b + u * join_waves < tile ? b + u * join_waves : tile - 1, v[u]);
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (b + u * join_waves < tile) {
#pragma unroll
            for (int c = 0; c < C; ++c) sum[c] += v[u][c];
          }
      }
#pragma unroll
      for (int c = 0; c < C; ++c) s_sum[w][c][lane] = sum[c];
      __syncthreads();
      if (w == 0 && mine > 0) {
        float last[C];
        read(heads, tile, last);
        out_t* const to = grad + static_cast<std::size_t>(row) * grad_pitch + own;
#pragma unroll
        for (int c = 0; c < C; ++c) {
          float v = s_sum[0][c][lane];
#pragma unroll
          for (int i = 1; i < join_waves; ++i) v += s_sum[i][c][lane];
          v += last[c];
          if (c < mine) to[c] = static_cast<out_t>(ADD ? __builtin_fmaf(scale, v, static_cast<float>(to[c])) : scale * v);
        }
      }
      __syncthreads();
    }
  }
}

/// One range of columns (at most max_columns).
template <typename type_t, typename out_t>
int launch_gradient_columns(hipStream_t stream, const int* keys, const int* positions, int tokens, int rows, const type_t* from,
                            std::size_t from_pitch, int dim, float scale, bool add, out_t* grad, std::size_t grad_pitch, void* workspace) {
  if (add && tokens <= small_tokens) {
    add_small<16, type_t, out_t><<<(dim + wave::size - 1) / wave::size, small_threads, 0, stream>>>(keys, positions, tokens, rows, from,
                                                                                                        from_pitch, dim, scale, grad, grad_pitch);
    return static_cast<int>(hipGetLastError());
  }
  const gradient_plan p = gradient_plan_for(lane_width<type_t, out_t>, tokens, dim);
  auto* const records = static_cast<tile_record*>(workspace);
  float* const heads = reinterpret_cast<float*>(static_cast<char*>(workspace) + gradient_records_bytes(p.tiles));
  float* const tails = heads + static_cast<std::size_t>(p.tiles) * dim;
  const unsigned int tile_groups = (static_cast<unsigned int>(p.tiles) * p.slabs + gradient_waves - 1) / gradient_waves;
  const int column_groups = (dim + 127) / 128;
  const int most = 2048 / column_groups > 1 ? 2048 / column_groups : 1;
  const dim3 join_grid(column_groups, p.tiles < most ? p.tiles : most);
  const bool whole_lines = (reinterpret_cast<std::uintptr_t>(grad) | (grad_pitch * sizeof(out_t)) | (dim * sizeof(out_t))) % 128 == 0;
  const clear_plan clear = clear_plan_for(rows, dim * sizeof(out_t), whole_lines);
  const auto run = [&](auto v_tag, auto add_tag) {
    constexpr int V = decltype(v_tag)::value;
    constexpr bool ADD = decltype(add_tag)::value;
    constexpr int U = ADD ? 4 : V * sizeof(type_t) > 8 ? 8 : 16;  // 8 to 16 KB of a wavefront's loads in flight
    const auto launch = [&](auto stream_tag) {
      const unsigned int grid = tile_groups + (ADD ? 0u : static_cast<unsigned int>(clear.groups));
      gradient<ADD, V, U, decltype(stream_tag)::value, type_t, out_t><<<grid, gradient_threads, 0, stream>>>(
          keys, positions, tokens, rows, from, from_pitch, dim, scale, grad, grad_pitch, p.tiles, p.items, p.slabs, tile_groups, clear, records, heads, tails);
    };
    if (!ADD && whole_lines) launch(std::bool_constant<!ADD && (V > 1)>{});  // (whole lines are wider than an access)
    else launch(std::false_type{});
    if (p.tiles > 1 && tokens >= whole_row)
      join<ADD, out_t><<<join_grid, join_threads, 0, stream>>>(records, heads, tails, p.tiles, dim, scale, grad, grad_pitch);
  };
  constexpr int V = lane_width<type_t, out_t>;
  if (dim < V) {
    if (add) run(std::integral_constant<int, 1>{}, std::true_type{});
    else run(std::integral_constant<int, 1>{}, std::false_type{});
  } else {
    if (add) run(std::integral_constant<int, V>{}, std::true_type{});
    else run(std::integral_constant<int, V>{}, std::false_type{});
  }
  return static_cast<int>(hipGetLastError());
}

template <typename type_t, typename out_t>
int launch_gradient(hipStream_t stream, const int* keys, const int* positions, int tokens, int rows, const type_t* from, std::size_t from_pitch,
                    int dim, float scale, bool add, out_t* grad, std::size_t grad_pitch, void* workspace) {
  if (rows == 0 || dim == 0 || (tokens == 0 && add)) return 0;
  return by_columns(dim, [&](int at, int cols) {
    return launch_gradient_columns<type_t, out_t>(stream, keys, positions, tokens, rows, from + at, from_pitch, cols, scale, add, grad + at, grad_pitch,
                                                  workspace);
  });
}

}  // namespace embedding
}  // namespace kernels
}  // namespace loops
