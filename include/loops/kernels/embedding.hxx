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

// ---- lookup -------------------------------------------------------------------------------------------------------------------
constexpr int lookup_threads = 256;

/**
 * A row is cut into `packets` = ceil(dim / V) packets of V values, the last one shifted back to end with the row (its overlap is
 * written twice, with the same values): any width and alignment moves in 16-byte accesses.  Packets of all rows are numbered through
 * and each thread takes U of them, a workgroup's width apart: consecutive lanes touch consecutive packets whatever the width.
 */
template <int V, int U, typename type_t, typename id_t>
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
      elements::store<V>(out + token[u] * out_pitch + column[u], v);
    }
  }
}

template <typename type_t, typename id_t>
int launch_lookup(hipStream_t stream, const type_t* table, std::size_t table_pitch, const id_t* ids, int tokens, int dim,
                  const group_ids::key_map& map, float scale, type_t* out, std::size_t out_pitch) {
  if (tokens == 0 || dim == 0) return 0;
  constexpr int V = elements::per_access<type_t>;
  const auto run = [&](auto v_tag, auto u_tag) {
    constexpr int W = decltype(v_tag)::value, U = decltype(u_tag)::value;
    const int packets = (dim + W - 1) / W;
    const unsigned long long all = static_cast<unsigned long long>(tokens) * packets;
    const unsigned long long grid = (all + lookup_threads * U - 1) / (lookup_threads * U);
    lookup<W, U, type_t, id_t><<<static_cast<unsigned int>(grid), lookup_threads, 0, stream>>>(table, table_pitch, ids, tokens, packets, dim, map,
                                                                                               scale, out, out_pitch);
  };
  const bool many = static_cast<unsigned long long>(tokens) * dim >= 512ull * lookup_threads * 4 * V;
  if (dim < V) run(std::integral_constant<int, 1>{}, std::integral_constant<int, 1>{});
  else if (many) run(std::integral_constant<int, V>{}, std::integral_constant<int, 4>{});
  else run(std::integral_constant<int, V>{}, std::integral_constant<int, 1>{});
  return static_cast<int>(hipGetLastError());
}

// ---- gradient -----------------------------------------------------------------------------------------------------------------
constexpr int gradient_threads = 256;
constexpr int gradient_waves = gradient_threads / wave::size;

/// Columns a wavefront covers.
template <typename type_t>
constexpr int slab = wave::size * elements::per_access<type_t>;

struct gradient_plan {
  int slabs;  ///< column slabs
  int items;  ///< merge items per tile
  int tiles;
};

/**
 * The tokens, sorted by row, and the rows' ends form one merge list (overwriting: an empty row costs a store, as a token costs a
 * load), or the tokens alone do (adding: rows without a token are not touched).  Equal tiles of that list, one wavefront per (tile,
 * slab of columns); a row of a hundred thousand tokens and a hundred thousand empty rows are the same work per wavefront.
 */
template <typename type_t>
gradient_plan gradient_plan_for(int tokens, int rows, int dim, bool add) {
  gradient_plan p;
  p.slabs = (dim + slab<type_t> - 1) / slab<type_t>;
  const long long total = static_cast<long long>(tokens) + (add ? 0 : rows);
  long long items = (total * p.slabs + 8191) / 8192;
  items = items < 8 ? 8 : items;
  p.items = static_cast<int>(items);
  p.tiles = static_cast<int>((total + items - 1) / items);
  return p;
}

/// What a tile leaves for the join: the row it finished that an earlier tile began, the row it began or continued and did not finish
/// (-1: none).
struct tile_record {
  int head_row;
  int tail_row;
};

/// Workspace: records[tiles], head[tiles][dim], tail[tiles][dim] (float).
inline std::size_t gradient_records_bytes(int tiles) { return (static_cast<std::size_t>(tiles) * sizeof(tile_record) + 255) & ~static_cast<std::size_t>(255); }
inline std::size_t gradient_workspace_bytes(const gradient_plan& p, int dim) {
  return gradient_records_bytes(p.tiles) + 2 * static_cast<std::size_t>(p.tiles) * dim * sizeof(float);
}

/// The number of tokens before merge position `at`: token j lies at j + key_j (the ends of the rows below key_j come first).  All
/// lanes search together, 64 probes a step.
__device__ __forceinline__ int tokens_before(const int* __restrict__ keys, int tokens, long long at) {
  int lo = 0, hi = tokens;  // answer in [lo, hi]: first j with j + key_j >= at
  while (hi > lo) {
    const int size = hi - lo;
    const int step = (size + wave::size - 1) / wave::size;
    const long long probe = static_cast<long long>(lo) + static_cast<long long>(wave::lane()) * step;
    bool below = false;
    if (probe < hi) below = probe + keys[probe] < at;
    const int n = __popcll(__ballot(below));  // probes below are a prefix of the lanes
    if (n == 0) return lo;
    const long long next_hi = static_cast<long long>(lo) + static_cast<long long>(n) * step;
    lo = lo + (n - 1) * step + 1;
    hi = next_hi < hi ? static_cast<int>(next_hi) : hi;
  }
  return lo;
}

/**
 * @tparam ADD  false: every row of grad is written (rows without tokens with zeros), true: rows with tokens are added to.
 * One wavefront per (tile, slab).  U gradient rows are in flight; ids and positions are wavefront-uniform (scalar loads).
 */
template <int V, int U, bool ADD, typename type_t, typename out_t>
__global__ void __launch_bounds__(gradient_threads)
gradient(const int* __restrict__ keys, const int* __restrict__ positions, const int tokens, const int rows, const type_t* __restrict__ from,
         const std::size_t from_pitch, const int dim, const float scale, out_t* __restrict__ grad, const std::size_t grad_pitch, const int tiles,
         const int items, const int slabs, tile_record* __restrict__ records, float* __restrict__ heads, float* __restrict__ tails) {
  const int unit = __builtin_amdgcn_readfirstlane(static_cast<int>(blockIdx.x) * gradient_waves + static_cast<int>(threadIdx.x) / wave::size);
  const int tile = unit / slabs;
  if (tile >= tiles) return;
  const int part = unit - tile * slabs;
  // the lane's columns; the last packet of a row is shifted back to end with it and stores its own columns only
  const int own = (part * wave::size + wave::lane()) * V;
  const bool active = own < dim;
  const bool whole = own + V <= dim;
  const int column = whole ? own : active ? dim - V : 0;
  const int skip = active ? own - column : V;

  const long long total = static_cast<long long>(tokens) + (ADD ? 0 : rows);
  const long long d0 = static_cast<long long>(tile) * items;
  const long long d1 = d0 + items < total ? d0 + items : total;
  int y = ADD ? static_cast<int>(d0) : __builtin_amdgcn_readfirstlane(tokens_before(keys, tokens, d0));
  const int before = y > 0 ? keys[y - 1] : -1;  // the row of the token before the tile
  int row = ADD ? (y < tokens ? keys[y] : rows) : static_cast<int>(d0 - y);
  bool open = before == row && row < rows;  // the row was begun by an earlier tile
  bool some = false;                        // tokens of this tile in the row
  int head_row = -1;

  const type_t* __restrict__ const base = from + column;
  float acc[V];
#pragma unroll
  for (int k = 0; k < V; ++k) acc[k] = 0.0f;

  const auto put_partial = [&](float* __restrict__ to) {
    if (active) {
      float* const at = to + static_cast<std::size_t>(tile) * dim;
#pragma unroll
      for (int k = 0; k < V; ++k)
        if (k >= skip) at[column + k] = acc[k];
    }
  };
  const auto finish = [&]() {  // the row's end
    if (open) {
      head_row = row;
      put_partial(heads);
      open = false;
    } else if (!ADD || some) {
      out_t* const at = grad + static_cast<std::size_t>(row) * grad_pitch + column;
      float v[V];
      if (whole) {
        if constexpr (ADD) {
#pragma unroll
          for (int k = 0; k < V; ++k) v[k] = __builtin_fmaf(scale, acc[k], static_cast<float>(at[k]));
        } else {
#pragma unroll
          for (int k = 0; k < V; ++k) v[k] = scale * acc[k];
        }
        elements::store<V>(at, v);
      } else if (active) {
#pragma unroll
        for (int k = 0; k < V; ++k)
          if (k >= skip) at[k] = static_cast<out_t>(ADD ? __builtin_fmaf(scale, acc[k], static_cast<float>(at[k])) : scale * acc[k]);
      }
    }
#pragma unroll
    for (int k = 0; k < V; ++k) acc[k] = 0.0f;
    some = false;
  };
  const auto clear = [&]() {  // a row without tokens
    out_t* const at = grad + static_cast<std::size_t>(row) * grad_pitch + column;
    const float zero[V] = {};
    if (whole) {
      elements::store<V>(at, zero);
    } else if (active) {
#pragma unroll
      for (int k = 0; k < V; ++k)
        if (k >= skip) at[k] = static_cast<out_t>(0.0f);
    }
  };

  // 64 tokens' keys and positions at a time, a token per lane; the tile's are a prefix of them
  for (;;) {
    const int j = y + wave::lane();
    int key = rows, position = 0;
    if (j < tokens) {
      key = keys[j];
      position = positions[j];
    }
    // (a position that group_ids did not write stays inside the array)
    if (static_cast<unsigned int>(position) >= static_cast<unsigned int>(tokens)) position = 0;
    const bool mine = key < rows && static_cast<long long>(j) + (ADD ? 0 : key) < d1;
    const int count = __popcll(__ballot(mine));
    for (int i = 0; i < count; i += U) {
      elements::packet_t<type_t, V> packet[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int at = i + u < count ? i + u : count - 1;
        packet[u] = elements::load<V>(base + static_cast<std::size_t>(__builtin_amdgcn_readlane(position, at)) * from_pitch);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (i + u < count) {
          const int k = __builtin_amdgcn_readlane(key, i + u);
          if (row < k) {
            finish();
            if constexpr (ADD) row = k;
            else
              for (++row; row < k; ++row) clear();
          }
          some = true;
#pragma unroll
          for (int c = 0; c < V; ++c) acc[c] += static_cast<float>(packet[u][c]);
        }
      }
    }
    y += count;
    if (count < wave::size) break;
  }
  // the rows that end in what is left of the tile
  bool unfinished;
  if constexpr (ADD) {
    unfinished = some && y < tokens && keys[y] == row;
    if (some && !unfinished) finish();
  } else {
    const int row1 = d1 - y < rows ? static_cast<int>(d1 - y) : rows;  // (tokens without a row lie behind all of them)
    if (row < row1) {
      finish();
      for (++row; row < row1; ++row) clear();
    }
    unfinished = some || open;
  }
  if (unfinished) put_partial(tails);
  if (part == 0 && wave::lane() == 0) records[tile] = tile_record{head_row, unfinished ? row : -1};
}

/**
 * The rows that more than one tile holds: sum of the tails of the tiles before, in a fixed order, and the finishing tile's head.
 * A workgroup covers 256 columns and walks over every gridDim.y-th run of 64 tiles; its four wavefronts share a row's tails out.
 */
template <bool ADD, typename out_t>
__global__ void __launch_bounds__(gradient_threads)
join(const tile_record* __restrict__ records, const float* __restrict__ heads, const float* __restrict__ tails, const int tiles, const int dim,
     const float scale, out_t* __restrict__ grad, const std::size_t grad_pitch) {
  constexpr int C = 4;  // columns per lane
  constexpr int U = 8;
  __shared__ float s_sum[gradient_waves][C][wave::size];
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
  for (int t0 = static_cast<int>(blockIdx.y) * wave::size; t0 < tiles; t0 += static_cast<int>(gridDim.y) * wave::size) {
    const int head = t0 + lane < tiles ? records[t0 + lane].head_row : -1;
    unsigned long long todo = __ballot(head >= 0);
    while (todo) {
      const int at = __builtin_ctzll(todo);
      todo &= todo - 1;
      const int tile = t0 + at;
      const int row = __builtin_amdgcn_readlane(head, at);
      int run = 0;  // tiles before this one that hold a part of the row
      for (;;) {
        const int t = tile - 1 - run - lane;
        const unsigned long long part = __ballot(t >= 0 && records[t < 0 ? 0 : t].tail_row == row);
        const int n = part == ~0ull ? wave::size : __builtin_ctzll(~part);
        run += n;
        if (n < wave::size) break;
      }
      float sum[C] = {0.0f, 0.0f, 0.0f, 0.0f};
      const int first = tile - run;
      for (int t = first + w; t < tile; t += gradient_waves * U) {
        float v[U][C];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int from = t + u * gradient_waves;
          read(tails, from < tile ? from : tile - 1, v[u]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (t + u * gradient_waves < tile) {
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
          for (int i = 1; i < gradient_waves; ++i) v += s_sum[i][c][lane];
          v += last[c];
          if (c < mine) to[c] = static_cast<out_t>(ADD ? __builtin_fmaf(scale, v, static_cast<float>(to[c])) : scale * v);
        }
      }
      __syncthreads();
    }
  }
}

template <typename type_t, typename out_t>
int launch_gradient(hipStream_t stream, const int* keys, const int* positions, int tokens, int rows, const type_t* from, std::size_t from_pitch,
                    int dim, float scale, bool add, out_t* grad, std::size_t grad_pitch, void* workspace) {
  if (rows == 0 || dim == 0 || (tokens == 0 && add)) return 0;
  const gradient_plan p = gradient_plan_for<type_t>(tokens, rows, dim, add);
  auto* const records = static_cast<tile_record*>(workspace);
  float* const heads = reinterpret_cast<float*>(static_cast<char*>(workspace) + gradient_records_bytes(p.tiles));
  float* const tails = heads + static_cast<std::size_t>(p.tiles) * dim;
  const unsigned int grid = (static_cast<unsigned int>(p.tiles) * p.slabs + gradient_waves - 1) / gradient_waves;
  const int column_groups = (dim + 255) / 256;
  const int tile_groups = (p.tiles + wave::size - 1) / wave::size;
  const int most = 1024 / column_groups > 1 ? 1024 / column_groups : 1;
  const dim3 join_grid(column_groups, tile_groups < most ? tile_groups : most);
  const auto run = [&](auto v_tag, auto add_tag) {
    constexpr int V = decltype(v_tag)::value;
    constexpr bool ADD = decltype(add_tag)::value;
    gradient<V, 8, ADD, type_t, out_t><<<grid, gradient_threads, 0, stream>>>(keys, positions, tokens, rows, from, from_pitch, dim, scale, grad,
                                                                             grad_pitch, p.tiles, p.items, p.slabs, records, heads, tails);
    if (p.tiles > 1)
      join<ADD, out_t><<<join_grid, gradient_threads, 0, stream>>>(records, heads, tails, p.tiles, dim, scale, grad, grad_pitch);
  };
  constexpr int V = elements::per_access<type_t>;
  if (dim < V) {
    if (add) run(std::integral_constant<int, 1>{}, std::true_type{});
    else run(std::integral_constant<int, 1>{}, std::false_type{});
  } else {
    if (add) run(std::integral_constant<int, V>{}, std::true_type{});
    else run(std::integral_constant<int, V>{}, std::false_type{});
  }
  return static_cast<int>(hipGetLastError());
}

}  // namespace embedding
}  // namespace kernels
}  // namespace loops
