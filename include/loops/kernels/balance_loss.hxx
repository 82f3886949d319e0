/**
 * @file balance_loss.hxx
 * @brief Tokens per expert and the balance loss of a router, with its gradient: column sums of the routing matrix R (tokens x experts,
 * `choices` ones per row) and of the probabilities.
 *
 *   p_t   = softmax(logits[t, :])                      c_e = #{(t, j) : chosen[t, j] = e, mask_t}          n = #{t : mask_t}
 *   loss  = a E sum_e (c_e / (n k)) (sum_t p_te / n)     d loss / d logits_te = a E / n * p_te (f_e - sum_j f_j p_tj),  f = c / (n k)
 *
 * (the counts are constants of the gradient, as the choice of experts has none).  A token whose mask does not hold takes no part and
 * its gradient is zero; n = 0 gives loss and gradient zero; a row of logits that are all -infinity has p = 0; choices outside [0, E)
 * are not counted.  The logits are read once in each direction and nothing of T x E is kept between them: the gradient computes its
 * softmax again, which costs no memory traffic.  Sums are held in float, counts in int.
 */
#pragma once

#include <cstddef>
#include <cstdint>
#include <type_traits>

#include <hip/hip_runtime.h>

#include <loops/util/elements.hxx>
#include <loops/util/wave.hxx>

namespace loops {
namespace kernels {
namespace balance {

constexpr int max_experts = 1024;
constexpr int threads = 1024;
constexpr int waves = threads / wave::size;
constexpr int max_groups = 512;  ///< workgroups whose partial sums the finish kernel adds up

namespace detail {

/// Which columns of a row a lane holds: K packets of V, packet k of lane l (of the G that share the row) is packet l + k G of the row.
/// The row's last packet is shifted back to end with it; its first `skip` elements belong to the packet before.
template <int V, int G, int K>
struct columns {
  int at[K];
  int skip[K];  ///< V: the packet lies past the row
  __device__ __forceinline__ explicit columns(int experts) {
    const int l = wave::lane() % G;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int own = (l + k * G) * V;
      const bool active = own < experts;
      at[k] = own + V <= experts ? own : active ? experts - V : 0;
      skip[k] = active ? own - at[k] : V;
    }
  }
};

template <int G>
__device__ __forceinline__ float row_max(float v) {
#pragma unroll
  for (int d = G / 2; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor(v, d, wave::size));
  return v;
}
template <int G>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int d = G / 2; d > 0; d >>= 1) v += __shfl_xor(v, d, wave::size);
  return v;
}

template <typename type_t, int V, int K>
struct row_packets {
  elements::packet_t<type_t, V> p[K];
};

template <int V, int G, int K, typename type_t>
__device__ __forceinline__ row_packets<type_t, V, K> read_row(const type_t* __restrict__ row, const columns<V, G, K>& c) {
  row_packets<type_t, V, K> r;
#pragma unroll
  for (int k = 0; k < K; ++k) r.p[k] = elements::load<V>(row + c.at[k]);
  return r;
}

/// The lane's part of softmax(row); columns that are not the lane's get 0.
template <int V, int G, int K, typename type_t>
__device__ __forceinline__ void softmax(const row_packets<type_t, V, K>& r, const columns<V, G, K>& c, float (&p)[K][V]) {
  constexpr float lowest = -__builtin_inff();
  float top = lowest;
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      p[k][e] = e >= c.skip[k] ? static_cast<float>(r.p[k][e]) : lowest;
      top = fmaxf(top, p[k][e]);
    }
  top = row_max<G>(top);
  if (top == lowest) top = 0.0f;  // nothing but -infinity (or NaN): exp gives 0 (NaN)
  float sum = 0.0f;
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      p[k][e] = __expf(p[k][e] - top);
      sum += p[k][e];
    }
  sum = row_sum<G>(sum);
  const float scale = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int e = 0; e < V; ++e) p[k][e] *= scale;
}

/// Sum over the workgroup, in a fixed order, in every thread (`scratch`: one float per wavefront).
__device__ __forceinline__ float block_sum(float v, float* __restrict__ scratch) {
  v = row_sum<wave::size>(v);
  const int w = static_cast<int>(threadIdx.x) / wave::size;
  if (wave::lane() == 0) scratch[w] = v;
  __syncthreads();
  float s = 0.0f;
  for (int i = 0; i < static_cast<int>(blockDim.x) / wave::size; ++i) s += scratch[i];
  __syncthreads();
  return s;
}

/// Adds the choices of tokens [begin, end) to `counts` (LDS).
template <typename id_t>
__device__ __forceinline__ void count_choices(const id_t* __restrict__ chosen, const unsigned char* __restrict__ mask, int choices, long long begin,
                                              long long end, int experts, int* __restrict__ counts) {
  const id_t* const from = chosen + begin * choices;
  const unsigned int n = static_cast<unsigned int>((end - begin) * choices);
  for (unsigned int i = threadIdx.x; i < n; i += blockDim.x) {
    const long long e = static_cast<long long>(from[i]);
    const bool counts_in = !mask || mask[begin + i / static_cast<unsigned int>(choices)] != 0;
    if (counts_in && e >= 0 && e < experts) atomicAdd(&counts[e], 1);
  }
}

}  // namespace detail

/// What the forward pass writes.
struct outputs {
  float* loss;         // [1]
  int* counts;         // [experts]
  float* probability;  // [experts]: mean over the counted tokens
  int* tokens;         // [1]: how many those are
};

namespace detail {
/// Thread e < experts brings column e's sum of probabilities and its count.
__device__ __forceinline__ void finish(float sum, int count, int tokens, int experts, int choices, float coefficient, const outputs& out,
                                       float* __restrict__ scratch) {
  const int e = threadIdx.x;
  const float per_token = tokens > 0 ? 1.0f / static_cast<float>(tokens) : 0.0f;
  float term = 0.0f;
  if (e < experts) {
    const float probability = sum * per_token;
    out.counts[e] = count;
    out.probability[e] = probability;
    term = static_cast<float>(count) * per_token / static_cast<float>(choices) * probability;
  }
  const float all = block_sum(term, scratch);
  if (threadIdx.x == 0) {
    *out.loss = coefficient * static_cast<float>(experts) * all;
    *out.tokens = tokens;
  }
}
}  // namespace detail

/**
 * Workgroup b reads tokens [b per, (b + 1) per): G lanes share a row, each keeps the sums of its own columns in registers over all of its
 * rows.  ONE: the only workgroup finishes as well; otherwise it leaves sums[b][experts], counts[b][experts], tokens[b].
 */
template <bool ONE, int V, int G, int K, int U, typename type_t, typename id_t>
__global__ void __launch_bounds__(threads)
forward(const type_t* __restrict__ logits, const std::size_t pitch, const id_t* __restrict__ chosen, const unsigned char* __restrict__ mask,
        const int tokens, const int experts, const int choices, const int per, const float coefficient, const outputs out,
        float* __restrict__ sums, int* __restrict__ counts, int* __restrict__ counted) {
  constexpr int rows_per_wave = wave::size / G;
  constexpr int rows_per_step = rows_per_wave * waves;
  __shared__ float s_sum[waves][K * G * V];
  __shared__ int s_count[max_experts];
  __shared__ float s_scratch[waves];
  __shared__ int s_tokens;
  const int tid = threadIdx.x;
  const int w = tid / wave::size;
  for (int e = tid; e < experts; e += threads) s_count[e] = 0;
  if (tid == 0) s_tokens = 0;
  __syncthreads();
  const long long begin = static_cast<long long>(blockIdx.x) * per;
  const long long end = begin + per < tokens ? begin + per : tokens;

  const detail::columns<V, G, K> cols(experts);
  float sum[K][V];
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int e = 0; e < V; ++e) sum[k][e] = 0.0f;
  int mine = 0;
  for (long long t0 = begin + w * rows_per_wave + wave::lane() / G; t0 < end; t0 += U * rows_per_step) {
    detail::row_packets<type_t, V, K> r[U];
    bool in[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long t = t0 + u * rows_per_step;
      in[u] = t < end;
      const long long from = in[u] ? t : t0;
      r[u] = detail::read_row<V, G, K>(logits + from * pitch, cols);
      if (mask) in[u] = in[u] && mask[from] != 0;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float p[K][V];
      detail::softmax<V, G, K>(r[u], cols, p);
      mine += in[u] ? 1 : 0;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e) sum[k][e] += in[u] ? p[k][e] : 0.0f;
    }
  }
  detail::count_choices(chosen, mask, choices, begin, end, experts, s_count);
  // rows of a wavefront, then wavefronts, always in the same order
#pragma unroll
  for (int d = G; d < wave::size; d <<= 1)
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < V; ++e) sum[k][e] += __shfl_xor(sum[k][e], d, wave::size);
  if (wave::lane() % G == 0 && mine) atomicAdd(&s_tokens, mine);
  if (wave::lane() < G) {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (e >= cols.skip[k]) s_sum[w][cols.at[k] + e] = sum[k][e];
  }
  __syncthreads();
  float total = 0.0f;
  if (tid < experts)
    for (int i = 0; i < waves; ++i) total += s_sum[i][tid];
  if constexpr (ONE) {
    detail::finish(total, tid < experts ? s_count[tid] : 0, s_tokens, experts, choices, coefficient, out, s_scratch);
  } else {
    if (tid < experts) {
      sums[static_cast<std::size_t>(blockIdx.x) * experts + tid] = total;
      counts[static_cast<std::size_t>(blockIdx.x) * experts + tid] = s_count[tid];
    }
    if (tid == 0) counted[blockIdx.x] = s_tokens;
  }
}

/// Adds the workgroups' sums up: 4 columns per thread, the workgroups dealt out to slices of the threads and added in a fixed order.
template <typename = void>
__global__ void __launch_bounds__(threads)
finish_forward(const float* __restrict__ sums, const int* __restrict__ counts, const int* __restrict__ counted, const int groups, const int experts,
               const int choices, const float coefficient, const outputs out) {
  constexpr int C = 4, U = 8;
  __shared__ float s_sum[threads * C];
  __shared__ int s_count[threads * C];
  __shared__ float s_scratch[waves];
  __shared__ int s_tokens;
  const int tid = threadIdx.x;
  int width = 1;  // threads per slice
  while (width * C < experts) width *= 2;
  const int slices = threads / width;
  const int column = tid % width * C;
  const int mine = column < experts ? (experts - column < C ? experts - column : C) : 0;
  if (tid == 0) s_tokens = 0;
  float sum[C] = {0.0f, 0.0f, 0.0f, 0.0f};
  int count[C] = {0, 0, 0, 0};
  if (mine > 0) {
    for (int b0 = tid / width; b0 < groups; b0 += slices * U) {
      float v[U][C];
      int n[U][C];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int b = b0 + u * slices < groups ? b0 + u * slices : b0;
        const std::size_t at = static_cast<std::size_t>(b) * experts + column;
        if (mine == C) {
          const auto x = elements::load<C>(sums + at);
          const auto y = elements::load<C>(counts + at);
#pragma unroll
          for (int c = 0; c < C; ++c) {
            v[u][c] = x[c];
            n[u][c] = y[c];
          }
        } else {
#pragma unroll
          for (int c = 0; c < C; ++c) {
            v[u][c] = c < mine ? sums[at + c] : 0.0f;
            n[u][c] = c < mine ? counts[at + c] : 0;
          }
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (b0 + u * slices < groups) {
#pragma unroll
          for (int c = 0; c < C; ++c) {
            sum[c] += v[u][c];
            count[c] += n[u][c];
          }
        }
    }
  }
#pragma unroll
  for (int c = 0; c < C; ++c) {
    s_sum[tid * C + c] = sum[c];
    s_count[tid * C + c] = count[c];
  }
  __syncthreads();
  if (tid < groups) atomicAdd(&s_tokens, counted[tid]);
  float total = 0.0f;
  int all = 0;
  if (tid < experts)
    for (int i = 0; i < slices; ++i) {
      total += s_sum[i * width * C + tid];
      all += s_count[i * width * C + tid];
    }
  __syncthreads();
  detail::finish(total, all, s_tokens, experts, choices, coefficient, out, s_scratch);
}

/// Gradient of the logits: G lanes share a row, which is read, turned into probabilities and written within the registers.
template <int V, int G, int K, int U, typename type_t>
__global__ void __launch_bounds__(256)
backward(const type_t* __restrict__ logits, const std::size_t pitch, const int* __restrict__ counts, const int* __restrict__ counted,
         const unsigned char* __restrict__ mask, const int tokens, const int experts, const int choices, const float coefficient,
         const float* __restrict__ grad_loss, type_t* __restrict__ grad, const std::size_t grad_pitch) {
  constexpr int rows_per_wave = wave::size / G;
  const detail::columns<V, G, K> cols(experts);
  const int n = *counted;
  const float per_token = n > 0 ? 1.0f / static_cast<float>(n) : 0.0f;
  const float scale = (grad_loss ? *grad_loss : 1.0f) * coefficient * static_cast<float>(experts) * per_token;
  const float share = per_token / static_cast<float>(choices);
  float weight[K][V];
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int e = 0; e < V; ++e) weight[k][e] = e >= cols.skip[k] ? static_cast<float>(counts[cols.at[k] + e]) * share : 0.0f;
  const long long stride = static_cast<long long>(gridDim.x) * (4 * rows_per_wave);
  for (long long t0 = static_cast<long long>(blockIdx.x) * (4 * rows_per_wave) + threadIdx.x / G; t0 < tokens; t0 += stride * U) {
    detail::row_packets<type_t, V, K> r[U];
    bool in[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long t = t0 + u * stride;
      const long long from = t < tokens ? t : t0;
      in[u] = !mask || mask[from] != 0;
      r[u] = detail::read_row<V, G, K>(logits + from * pitch, cols);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float p[K][V];
      detail::softmax<V, G, K>(r[u], cols, p);
      float dot = 0.0f;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e) dot += p[k][e] * weight[k][e];
      dot = detail::row_sum<G>(dot);
      const long long t = t0 + u * stride;
      if (t < tokens) {
        type_t* const to = grad + t * grad_pitch;
#pragma unroll
        for (int k = 0; k < K; ++k) {
          float g[V];
#pragma unroll
          for (int e = 0; e < V; ++e) g[e] = in[u] ? p[k][e] * (weight[k][e] - dot) * scale : 0.0f;
          if (cols.skip[k] == 0) {
            elements::store<V>(to + cols.at[k], g);
          } else {
#pragma unroll
            for (int e = 0; e < V; ++e)
              if (e >= cols.skip[k]) to[cols.at[k] + e] = static_cast<type_t>(g[e]);
          }
        }
      }
    }
  }
}

// ---- counts alone ---------------------------------------------------------------------------------------------------------------
/// Workgroup b counts the choices of tokens [b per, (b + 1) per) into counts[b][experts].
template <typename id_t>
__global__ void __launch_bounds__(threads)
count_experts(const id_t* __restrict__ chosen, const unsigned char* __restrict__ mask, const int tokens, const int choices, const int experts,
              const int per, int* __restrict__ counts) {
  __shared__ int s_count[max_experts];
  for (int e = threadIdx.x; e < experts; e += threads) s_count[e] = 0;
  __syncthreads();
  const long long begin = static_cast<long long>(blockIdx.x) * per;
  const long long end = begin + per < tokens ? begin + per : tokens;
  detail::count_choices(chosen, mask, choices, begin, end, experts, s_count);
  __syncthreads();
  for (int e = threadIdx.x; e < experts; e += threads) counts[static_cast<std::size_t>(blockIdx.x) * experts + e] = s_count[e];
}

/// counts[e] = sum over the workgroups: 64 experts per workgroup, 16 threads each.
template <typename = void>
__global__ void __launch_bounds__(threads) finish_counts(const int* __restrict__ partial, const int groups, const int experts, int* __restrict__ counts) {
  __shared__ int s_count[waves][wave::size];
  const int e = static_cast<int>(blockIdx.x) * wave::size + wave::lane();
  const int w = static_cast<int>(threadIdx.x) / wave::size;
  int sum = 0;
  if (e < experts) {
#pragma unroll 8
    for (int b = w; b < groups; b += waves) sum += partial[static_cast<std::size_t>(b) * experts + e];
  }
  s_count[w][wave::lane()] = sum;
  __syncthreads();
  if (w == 0 && e < experts) {
    for (int i = 1; i < waves; ++i) sum += s_count[i][wave::lane()];
    counts[e] = sum;
  }
}

// ---- launches -------------------------------------------------------------------------------------------------------------------
struct groups_t {
  int groups;
  int per;  ///< tokens per workgroup
};
inline groups_t share_out(int tokens, long long work_per_token, long long least, int most) {
  long long groups = (tokens * work_per_token + least - 1) / least;
  groups = groups < 1 ? 1 : groups > most ? most : groups;
  groups_t g;
  g.per = static_cast<int>((tokens + groups - 1) / groups);
  if (g.per < 1) g.per = 1;
  g.groups = (tokens + g.per - 1) / g.per;
  if (g.groups < 1) g.groups = 1;
  return g;
}
/// One workgroup up to 32 768 logits.
inline groups_t forward_groups(int tokens, int experts) { return share_out(tokens, experts, static_cast<long long>(tokens) * experts <= 32768 ? 32768 : 16384, max_groups); }
inline groups_t count_groups(int tokens, int choices) { return share_out(tokens, choices, 16384, max_groups); }

inline std::size_t forward_workspace_bytes(int tokens, int experts) {
  const groups_t g = forward_groups(tokens, experts);
  return g.groups == 1 ? 0 : static_cast<std::size_t>(g.groups) * (2 * static_cast<std::size_t>(experts) + 1) * 4;
}
inline std::size_t count_workspace_bytes(int tokens, int choices, int experts) {
  const groups_t g = count_groups(tokens, choices);
  return g.groups == 1 ? 0 : static_cast<std::size_t>(g.groups) * experts * sizeof(int);
}

/// Calls f(V, G, K) as integral constants: lanes per row and packets per lane for rows of `experts` values.
template <typename type_t, typename F>
void with_shape(int experts, F&& f) {
  constexpr int V = elements::per_access<type_t>;
  using one = std::integral_constant<int, 1>;
  using v = std::integral_constant<int, V>;
  const int packets = (experts + V - 1) / V;
  if (experts < V) f(one{}, std::integral_constant<int, 8>{}, one{});
  else if (packets <= 8) f(v{}, std::integral_constant<int, 8>{}, one{});
  else if (packets <= 16) f(v{}, std::integral_constant<int, 16>{}, one{});
  else if (packets <= 32) f(v{}, std::integral_constant<int, 32>{}, one{});
  else if (packets <= 64) f(v{}, std::integral_constant<int, 64>{}, one{});
  else if (packets <= 128) f(v{}, std::integral_constant<int, 64>{}, std::integral_constant<int, 2>{});
  else if constexpr (sizeof(type_t) == 4) f(v{}, std::integral_constant<int, 64>{}, std::integral_constant<int, 4>{});
}

template <typename type_t, typename id_t>
int launch_forward(hipStream_t stream, const type_t* logits, std::size_t pitch, const id_t* chosen, const unsigned char* mask, int tokens, int experts,
                   int choices, float coefficient, const outputs& out, void* workspace) {
  const groups_t g = forward_groups(tokens, experts);
  float* const sums = static_cast<float*>(workspace);
  int* const counts = reinterpret_cast<int*>(sums + static_cast<std::size_t>(g.groups) * experts);
  int* const counted = counts + static_cast<std::size_t>(g.groups) * experts;
  with_shape<type_t>(experts, [&](auto v, auto lanes, auto k) {
    constexpr int V = decltype(v)::value, G = decltype(lanes)::value, K = decltype(k)::value, U = K == 1 ? 2 : 1;
    if (g.groups == 1)
      forward<true, V, G, K, U, type_t, id_t><<<1, threads, 0, stream>>>(logits, pitch, chosen, mask, tokens, experts, choices, g.per, coefficient, out,
                                                                       nullptr, nullptr, nullptr);
    else
      forward<false, V, G, K, U, type_t, id_t><<<g.groups, threads, 0, stream>>>(logits, pitch, chosen, mask, tokens, experts, choices, g.per,
                                                                               coefficient, out, sums, counts, counted);
  });
  if (g.groups > 1) finish_forward<><<<1, threads, 0, stream>>>(sums, counts, counted, g.groups, experts, choices, coefficient, out);
  return static_cast<int>(hipGetLastError());
}

template <typename type_t>
int launch_backward(hipStream_t stream, const type_t* logits, std::size_t pitch, const int* counts, const int* counted, const unsigned char* mask,
                    int tokens, int experts, int choices, float coefficient, const float* grad_loss, type_t* grad, std::size_t grad_pitch) {
  if (tokens == 0) return 0;
  with_shape<type_t>(experts, [&](auto v, auto lanes, auto k) {
    constexpr int V = decltype(v)::value, G = decltype(lanes)::value, K = decltype(k)::value, U = K == 1 ? 2 : 1;
    constexpr int rows = 4 * (wave::size / G);
    const long long groups = (static_cast<long long>(tokens) + rows - 1) / rows;
    const unsigned int grid = static_cast<unsigned int>(groups < 2048 ? groups : 2048);
    backward<V, G, K, U, type_t><<<grid, 256, 0, stream>>>(logits, pitch, counts, counted, mask, tokens, experts, choices, coefficient, grad_loss, grad,
                                                          grad_pitch);
  });
  return static_cast<int>(hipGetLastError());
}

template <typename id_t>
int launch_counts(hipStream_t stream, const id_t* chosen, const unsigned char* mask, int tokens, int choices, int experts, int* counts, void* workspace) {
  const groups_t g = count_groups(tokens, choices);
  int* const partial = g.groups == 1 ? counts : static_cast<int*>(workspace);
  count_experts<id_t><<<g.groups, threads, 0, stream>>>(chosen, mask, tokens, choices, experts, g.per, partial);
  if (g.groups > 1)
    finish_counts<><<<(experts + wave::size - 1) / wave::size, threads, 0, stream>>>(partial, g.groups, experts, counts);
  return static_cast<int>(hipGetLastError());
}

}  // namespace balance
}  // namespace kernels
}  // namespace loops
