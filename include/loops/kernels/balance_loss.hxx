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
/// FULL: the row is G K V columns.  Otherwise its last packet is shifted back to end with it, and the first `skip` elements of that belong
/// to the packet before.
template <bool FULL, int V, int G, int K>
struct columns {
  int at[K];
  int skip[K];  ///< V: the packet lies past the row
  __device__ __forceinline__ explicit columns(int experts) {
    const int l = wave::lane() % G;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int own = (l + k * G) * V;
      const bool active = FULL || own < experts;
      at[k] = FULL || own + V <= experts ? own : active ? experts - V : 0;
      skip[k] = active ? own - at[k] : V;
    }
  }
  __device__ __forceinline__ bool mine(int k, int e) const { return FULL || e >= skip[k]; }
};

/// v of the lane that differs in bit log2(D) of its number where the lanes below D agree: a step of a reduction over 2 D lanes.  Within
/// 16 lanes by DPP, beyond by gfx950's row swaps: no LDS traffic.
template <int D>
__device__ __forceinline__ void partner(float v, float& a, float& b) {
  const int i = __builtin_bit_cast(int, v);
  if constexpr (D < 16) {
    constexpr int ctrl = D == 1 ? 0xB1 : D == 2 ? 0x4E : D == 4 ? 0x141 : 0x140;  // quad_perm [1,0,3,2], [2,3,0,1], row_half_mirror, row_mirror
    a = v;
    b = __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(i, i, ctrl, 0xF, 0xF, true));
  } else if constexpr (D == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(i, i, false, false);
    a = __builtin_bit_cast(float, static_cast<int>(r[0]));
    b = __builtin_bit_cast(float, static_cast<int>(r[1]));
  } else {
    const auto r = __builtin_amdgcn_permlane32_swap(i, i, false, false);
    a = __builtin_bit_cast(float, static_cast<int>(r[0]));
    b = __builtin_bit_cast(float, static_cast<int>(r[1]));
  }
}
/// Over G adjacent lanes, the result in all of them.
template <int G, typename F>
__device__ __forceinline__ float row_reduce(float v, F&& f) {
  float a, b;
  const auto step = [&](auto d) {
    if constexpr (decltype(d)::value < G) {
      partner<decltype(d)::value>(v, a, b);
      v = f(a, b);
    }
  };
  step(std::integral_constant<int, 1>{});
  step(std::integral_constant<int, 2>{});
  step(std::integral_constant<int, 4>{});
  step(std::integral_constant<int, 8>{});
  step(std::integral_constant<int, 16>{});
  step(std::integral_constant<int, 32>{});
  return v;
}
template <int G>
__device__ __forceinline__ float row_max(float v) {
  return row_reduce<G>(v, [](float a, float b) { return fmaxf(a, b); });
}
template <int G>
__device__ __forceinline__ float row_sum(float v) {
  return row_reduce<G>(v, [](float a, float b) { return a + b; });
}

template <typename type_t, int V, int K>
struct row_packets {
  elements::packet_t<type_t, V> p[K];
};

template <typename type_t, typename cols_t, int V, int K>
__device__ __forceinline__ void read_row(const type_t* __restrict__ row, const cols_t& c, row_packets<type_t, V, K>& r) {
#pragma unroll
  for (int k = 0; k < K; ++k) r.p[k] = elements::load<V>(row + c.at[k]);
}

/// exp(d) for d <= 0 as 2^(d log2(e)), the hardware's exponential (1 ulp; results below 2^-126 are 0).  The product's rounding alone would be an error
/// of up to |d| / 2 ulp.  FINE: what the product h leaves out, l = d log2(e) - h from a log2(e) in two parts, comes back as the factor 2^l = 1 + l ln 2
/// (|l| < 2^-17).  Where the exponential is 0, l may be infinite or NaN and is bounded for its product with 0.
/// Float logits are FINE (16 384 x 128: forward 11.8 us without it, 12.4 with, backward 6.0, 6.6; 262 139 x 256: 55, 65, and 97, 98); halves and
/// bfloat16 save the five instructions per element, as a store rounds their gradient to 2^-12 or 2^-9 anyway.
template <bool FINE>
__device__ __forceinline__ float exponential(float d) {
  constexpr float log2e = 1.44269504088896340736f, rest = static_cast<float>(1.44269504088896340736 - static_cast<double>(log2e)), ln2 = 0.693147180559945309417f;
  const float h = d * log2e;
  const float p = __builtin_amdgcn_exp2f(h);
  if constexpr (!FINE) return p;
  const float l = __builtin_fmaf(d, rest, __builtin_fmaf(d, log2e, -h));
  return __builtin_fmaf(p * __builtin_amdgcn_fmed3f(l, -1.0f, 1.0f), ln2, p);
}

/// p = exp(row - its maximum) in the lane's columns (0 in columns that are not its own); returns the factor that makes it the softmax.  A row
/// that takes no part is read as zeros and has the factor 0: what it holds (NaN) reaches nothing.
/// (x - top, then times log2(e): one fma of x would save an instruction, but its rounding of top log2(e) is not small in a row at the type's
/// lowest value.)
template <int G, typename cols_t, typename type_t, int V, int K>
__device__ __forceinline__ float exponentials(row_packets<type_t, V, K>& r, bool in, const cols_t& c, float (&p)[K][V]) {
  constexpr float lowest = -__builtin_inff();
  float top = lowest;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if (!in) r.p[k] = elements::packet_t<type_t, V>{};
#pragma unroll
    for (int e = 0; e < V; ++e) {
      p[k][e] = c.mine(k, e) ? static_cast<float>(r.p[k][e]) : lowest;
      top = fmaxf(top, p[k][e]);
    }
  }
  top = row_max<G>(top);
  if (top == lowest) top = 0.0f;  // nothing but -infinity (or NaN): exp gives 0 (NaN)
  float sum = 0.0f;
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      p[k][e] = exponential<sizeof(type_t) == 4>(p[k][e] - top);
      sum += p[k][e];
    }
  sum = row_sum<G>(sum);
  float factor = __builtin_amdgcn_rcpf(sum);
  if constexpr (sizeof(type_t) == 4) factor = __builtin_fmaf(__builtin_fmaf(-sum, factor, 1.0f), factor, factor);  // (a row: no matter of time)
  return !in || sum == 0.0f ? 0.0f : factor;
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
  constexpr unsigned int U = 4;  // reads in flight
  for (unsigned int i = threadIdx.x; i < n; i += U * blockDim.x) {
    long long e[U];
    unsigned char counts_in[U];
#pragma unroll
    for (unsigned int u = 0; u < U; ++u) {
      const unsigned int at = i + u * blockDim.x < n ? i + u * blockDim.x : i;
      e[u] = static_cast<long long>(from[at]);
      counts_in[u] = mask ? mask[begin + at / static_cast<unsigned int>(choices)] : 1;
    }
#pragma unroll
    for (unsigned int u = 0; u < U; ++u)
      if (i + u * blockDim.x < n && counts_in[u] != 0 && e[u] >= 0 && e[u] < experts) atomicAdd(&counts[e[u]], 1);
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
/// Writes column e's outputs and returns its term of the loss.  Factors of a whole result are products of double, rounded once.
__device__ __forceinline__ float finish_column(int e, float sum, int count, int tokens, int experts, int choices, const outputs& out) {
  if (e >= experts) return 0.0f;
  const double per_token = tokens > 0 ? 1.0 / tokens : 0.0;
  const double probability = sum * per_token;
  out.counts[e] = count;
  out.probability[e] = static_cast<float>(probability);
  return static_cast<float>(count * per_token / choices * probability);
}
}  // namespace detail

/// Floats (ints) between the partial sums (counts) of two workgroups: whole groups of columns of the finish kernel.
__host__ __device__ constexpr int partial_pitch(int experts) { return (experts + wave::size - 1) / wave::size * wave::size; }

/**
 * Workgroup b reads tokens [b per, (b + 1) per): G lanes share a row, each keeps the sums of its own columns in registers over all of its
 * rows.  262 139 x 256 bf16 with 8 choices each: 33 us, 4.6 TB/s of logits and ids (float: at `exponential`); the exponentials of a row and its
 * reductions share the time with the reads.  ONE: the only workgroup finishes as well; otherwise it leaves sums[b], counts[b] (rows of partial_pitch) and counted[b].
 */
template <bool ONE, bool FULL, int V, int G, int K, int U, typename type_t, typename id_t>
__global__ void __launch_bounds__(threads)
forward(const type_t* __restrict__ logits, const std::size_t pitch, const id_t* __restrict__ chosen, const unsigned char* __restrict__ mask,
        const int tokens, const int experts, const int choices, const int per, const float coefficient, const outputs out,
        float* __restrict__ sums, int* __restrict__ counts, int* __restrict__ counted, int* __restrict__ finished) {
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

  detail::count_choices(chosen, mask, choices, begin, end, experts, s_count);
  const detail::columns<FULL, V, G, K> cols(experts);
  float sum[K][V];
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int e = 0; e < V; ++e) sum[k][e] = 0.0f;
  int mine = 0;
  const int last = static_cast<int>(end);
  int t0 = static_cast<int>(begin) + w * rows_per_wave + wave::lane() / G;
  const type_t* __restrict__ row = logits + static_cast<std::size_t>(t0) * pitch;
  const std::size_t step = static_cast<std::size_t>(rows_per_step) * pitch;
  for (; t0 < last; t0 += U * rows_per_step, row += U * step) {
    detail::row_packets<type_t, V, K> r[U];
    unsigned char counts_in[U];
    bool in[U];
#pragma unroll
    for (int u = 0; u < U; ++u) counts_in[u] = 1;
    if (mask) {
#pragma unroll
      for (int u = 0; u < U; ++u) counts_in[u] = mask[t0 + u * rows_per_step < last ? t0 + u * rows_per_step : t0];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) detail::read_row(t0 + u * rows_per_step < last ? row + u * step : row, cols, r[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) in[u] = t0 + u * rows_per_step < last && counts_in[u] != 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float p[K][V];
      const float scale = detail::exponentials<G>(r[u], in[u], cols, p);
      mine += in[u] ? 1 : 0;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e) sum[k][e] = __builtin_fmaf(p[k][e], scale, sum[k][e]);
    }
  }
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
        if (cols.mine(k, e)) s_sum[w][cols.at[k] + e] = sum[k][e];
  }
  __syncthreads();
  float total = 0.0f;
  if (tid < experts)
    for (int i = 0; i < waves; ++i) total += s_sum[i][tid];
  if constexpr (ONE) {
    const float term = detail::finish_column(tid, total, tid < experts ? s_count[tid] : 0, s_tokens, experts, choices, out);
    const float loss = detail::block_sum(term, s_scratch);
    if (tid == 0) {
      *out.loss = static_cast<float>(static_cast<double>(coefficient) * experts * loss);
      *out.tokens = s_tokens;
    }
  } else {
    if (tid < experts) {
      sums[static_cast<std::size_t>(blockIdx.x) * partial_pitch(experts) + tid] = total;
      counts[static_cast<std::size_t>(blockIdx.x) * partial_pitch(experts) + tid] = s_count[tid];
    }
    if (tid == 0) {
      counted[blockIdx.x] = s_tokens;
      if (blockIdx.x == 0) *finished = 0;
    }
  }
}

/**
 * Adds the workgroups' sums up, in a fixed order: a workgroup takes 16 columns, 4 per thread, and deals the `groups` out to 256 slices of
 * its threads (512 x 256: 8.0 us at 64 columns per workgroup, 7.6 at 16; launch, one round of reads and the two trips of the count).  Its part of the loss
 * goes into parts[blockIdx.x]; the workgroup that counts itself last in *finished (0 at the start: the forward kernel cleared it) adds the
 * parts up.  No workgroup waits for another.
 */
constexpr int finish_columns = 16;
static_assert(max_experts / finish_columns <= wave::size, "a lane per part of the loss");

template <typename = void>
__global__ void __launch_bounds__(threads)
finish_forward(const float* __restrict__ sums, const int* __restrict__ counts, const int* __restrict__ counted, const int groups, const int experts,
               const int choices, const float coefficient, const outputs out, float* __restrict__ parts, int* __restrict__ finished) {
  constexpr int C = 4;
  constexpr int width = finish_columns / C;  // threads across the columns
  constexpr int slices = threads / width;
  constexpr int apart = finish_columns + C;  // (rows of LDS, a few banks apart)
  __shared__ float s_sum[slices * apart];
  __shared__ int s_count[slices * apart];
  __shared__ int s_tokens;
  const int tid = threadIdx.x;
  const int slice = tid / width;
  const int local = tid % width * C;
  if (tid == 0) s_tokens = 0;
  typedef float real_t __attribute__((ext_vector_type(C)));
  typedef int whole_t __attribute__((ext_vector_type(C)));
  real_t sum = {0.0f, 0.0f, 0.0f, 0.0f};
  whole_t count = {0, 0, 0, 0};
  const int pitch = partial_pitch(experts);  // (columns past the last expert are read, and dropped)
  const int from = static_cast<int>(blockIdx.x) * finish_columns + local;
  for (int b = slice; b < groups; b += slices) {
    const std::size_t at = static_cast<std::size_t>(b) * pitch + from;
    sum += *reinterpret_cast<const real_t*>(sums + at);
    count += *reinterpret_cast<const whole_t*>(counts + at);
  }
#pragma unroll
  for (int c = 0; c < C; ++c) {
    s_sum[slice * apart + local + c] = sum[c];
    s_count[slice * apart + local + c] = count[c];
  }
  __syncthreads();
  if (tid < groups) atomicAdd(&s_tokens, counted[tid]);
  // 256 slices to 64 (one column per thread), to 16 (4 of a wavefront's), to one
  constexpr int per_wave = slices / waves;
  constexpr int rows = wave::size / finish_columns;
  const int w = tid / wave::size, column = tid % finish_columns, row = wave::lane() / finish_columns;
  float total = 0.0f;
  int all = 0;
#pragma unroll
  for (int i = row; i < per_wave; i += rows) {
    total += s_sum[(w * per_wave + i) * apart + column];
    all += s_count[(w * per_wave + i) * apart + column];
  }
  const auto fold = [&]() {
#pragma unroll
    for (int d = finish_columns; d < wave::size; d <<= 1) {
      total += __shfl_xor(total, d, wave::size);
      all += __shfl_xor(all, d, wave::size);
    }
  };
  fold();
  __syncthreads();
  if (row == 0) {
    s_sum[w * apart + column] = total;
    s_count[w * apart + column] = all;
  }
  __syncthreads();
  if (w == 0) {
    total = 0.0f;
    all = 0;
#pragma unroll
    for (int i = row; i < waves; i += rows) {
      total += s_sum[i * apart + column];
      all += s_count[i * apart + column];
    }
    fold();
    const int e = row == 0 ? static_cast<int>(blockIdx.x) * finish_columns + column : experts;
    const float part = detail::row_sum<wave::size>(detail::finish_column(e, total, all, s_tokens, experts, choices, out));
    int before = 0;
    if (wave::lane() == 0) {
      __hip_atomic_store(parts + blockIdx.x, part, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      before = __hip_atomic_fetch_add(finished, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
    }
    if (__builtin_amdgcn_readfirstlane(before) == static_cast<int>(gridDim.x) - 1) {
      const int lane = wave::lane();
      const float loss = detail::row_sum<wave::size>(
          lane < static_cast<int>(gridDim.x) ? __hip_atomic_load(parts + lane, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0.0f);
      if (lane == 0) {
        *out.loss = static_cast<float>(static_cast<double>(coefficient) * experts * loss);
        *out.tokens = s_tokens;
      }
    }
  }
}

/// Gradient of the logits: G lanes share a row, which is read, turned into probabilities and written within the registers.  HBM bounds it:
/// 262 139 x 256 bf16 in 42 us, 6.3 TB/s.
template <bool FULL, int V, int G, int K, int U, typename type_t>
__global__ void __launch_bounds__(256)
backward(const type_t* __restrict__ logits, const std::size_t pitch, const int* __restrict__ counts, const int* __restrict__ counted,
         const unsigned char* __restrict__ mask, const int tokens, const int experts, const int choices, const float coefficient,
         const float* __restrict__ grad_loss, type_t* __restrict__ grad, const std::size_t grad_pitch) {
  constexpr int rows_per_wave = wave::size / G;
  const detail::columns<FULL, V, G, K> cols(experts);
  const int n = *counted;
  const double per_token = n > 0 ? 1.0 / n : 0.0;  // (factors of the whole gradient: rounded once, as products)
  const float scale = static_cast<float>(static_cast<double>(grad_loss ? *grad_loss : 1.0f) * coefficient * experts * per_token);
  const double share = per_token / choices;
  float weight[K][V];
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int e = 0; e < V; ++e) weight[k][e] = cols.mine(k, e) ? static_cast<float>(counts[cols.at[k] + e] * share) : 0.0f;
  const unsigned int count = static_cast<unsigned int>(tokens);
  const unsigned int stride = gridDim.x * (4 * rows_per_wave);
  unsigned int t0 = blockIdx.x * (4 * rows_per_wave) + threadIdx.x / G;
  const type_t* __restrict__ row = logits + static_cast<std::size_t>(t0) * pitch;
  type_t* __restrict__ to_row = grad + static_cast<std::size_t>(t0) * grad_pitch;
  const std::size_t step = static_cast<std::size_t>(stride) * pitch, to_step = static_cast<std::size_t>(stride) * grad_pitch;
  for (; t0 < count; t0 += stride * U, row += U * step, to_row += U * to_step) {
    detail::row_packets<type_t, V, K> r[U];
    unsigned char counts_in[U];
    bool in[U];
#pragma unroll
    for (int u = 0; u < U; ++u) counts_in[u] = 1;
    if (mask) {
#pragma unroll
      for (int u = 0; u < U; ++u) counts_in[u] = mask[t0 + u * stride < count ? t0 + u * stride : t0];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) detail::read_row(t0 + u * stride < count ? row + u * step : row, cols, r[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) in[u] = counts_in[u] != 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float p[K][V];
      const float factor = detail::exponentials<G>(r[u], in[u], cols, p);
      float dot = 0.0f;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e) dot = __builtin_fmaf(p[k][e], weight[k][e], dot);
      dot = detail::row_sum<G>(dot) * factor;
      const float by = factor == 0.0f ? 0.0f : factor * scale;  // (also for an upstream gradient that is not finite)
      if (t0 + u * stride < count) {
        type_t* const to = to_row + u * to_step;
#pragma unroll
        for (int k = 0; k < K; ++k) {
          float g[V];
#pragma unroll
          for (int e = 0; e < V; ++e) g[e] = p[k][e] * by * (weight[k][e] - dot);
          if (FULL || cols.skip[k] == 0) {
            elements::store<V>(to + cols.at[k], g);
          } else {
#pragma unroll
            for (int e = 0; e < V; ++e)
              if (cols.mine(k, e)) to[cols.at[k] + e] = static_cast<type_t>(g[e]);
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
  g.groups = static_cast<int>((static_cast<long long>(tokens) + g.per - 1) / g.per);  // (per is 4 million near 2^31 tokens)
  if (g.groups < 1) g.groups = 1;
  return g;
}
/// One workgroup up to 32 768 logits: without the second launch 256 x 128 takes 6.8 us (8.0 with it), 512 x 128 10.7 (9.0).
inline groups_t forward_groups(int tokens, int experts) { return share_out(tokens, experts, static_cast<long long>(tokens) * experts <= 32768 ? 32768 : 16384, max_groups); }
inline groups_t count_groups(int tokens, int choices) { return share_out(tokens, choices, 4096, max_groups); }

inline int finish_groups(int experts) { return (experts + finish_columns - 1) / finish_columns; }
/// sums[groups][pitch], counts[groups][pitch], counted[groups], parts[finish_groups], finished[1].
inline std::size_t forward_workspace_bytes(int tokens, int experts) {
  const groups_t g = forward_groups(tokens, experts);
  return g.groups == 1 ? 0 : (static_cast<std::size_t>(g.groups) * (2 * static_cast<std::size_t>(partial_pitch(experts)) + 1) + finish_groups(experts) + 1) * 4;
}
inline std::size_t count_workspace_bytes(int tokens, int choices, int experts) {
  const groups_t g = count_groups(tokens, choices);
  return g.groups == 1 ? 0 : static_cast<std::size_t>(g.groups) * experts * sizeof(int);
}

/// Calls f(FULL, V, G, K) as integral constants: lanes per row and packets per lane for rows of `experts` values.
template <typename type_t, typename F>
void with_shape(int experts, F&& f) {
  constexpr int V = elements::per_access<type_t>;
  using one = std::integral_constant<int, 1>;
  const auto with = [&](auto v, auto lanes, auto k) {
    if (experts == decltype(v)::value * decltype(lanes)::value * decltype(k)::value) f(std::true_type{}, v, lanes, k);
    else f(std::false_type{}, v, lanes, k);
  };
  const std::integral_constant<int, V> v{};
  const int packets = (experts + V - 1) / V;
  if (experts < V) f(std::false_type{}, one{}, std::integral_constant<int, 8>{}, one{});
  else if (packets <= 8) with(v, std::integral_constant<int, 8>{}, one{});
  else if (packets <= 16) with(v, std::integral_constant<int, 16>{}, one{});
  else if (packets <= 32) with(v, std::integral_constant<int, 32>{}, one{});
  else if (packets <= 64) with(v, std::integral_constant<int, 64>{}, one{});
  else if (packets <= 128) with(v, std::integral_constant<int, 64>{}, std::integral_constant<int, 2>{});
  else if constexpr (sizeof(type_t) == 4) with(v, std::integral_constant<int, 64>{}, std::integral_constant<int, 4>{});
}

template <typename type_t, typename id_t>
int launch_forward(hipStream_t stream, const type_t* logits, std::size_t pitch, const id_t* chosen, const unsigned char* mask, int tokens, int experts,
                   int choices, float coefficient, const outputs& out, void* workspace) {
  const groups_t g = forward_groups(tokens, experts);
  float* const sums = static_cast<float*>(workspace);
  int* const counts = reinterpret_cast<int*>(sums + static_cast<std::size_t>(g.groups) * partial_pitch(experts));
  int* const counted = counts + static_cast<std::size_t>(g.groups) * partial_pitch(experts);
  float* const parts = reinterpret_cast<float*>(counted + g.groups);
  int* const finished = reinterpret_cast<int*>(parts + finish_groups(experts));
  with_shape<type_t>(experts, [&](auto full, auto v, auto lanes, auto k) {
    constexpr bool FULL = decltype(full)::value;
    constexpr int V = decltype(v)::value, G = decltype(lanes)::value, K = decltype(k)::value, U = K == 1 ? 2 : 1;
    if (g.groups == 1)
      forward<true, FULL, V, G, K, U, type_t, id_t><<<1, threads, 0, stream>>>(logits, pitch, chosen, mask, tokens, experts, choices, g.per, coefficient, out,
                                                                       nullptr, nullptr, nullptr, nullptr);
    else
      forward<false, FULL, V, G, K, U, type_t, id_t><<<g.groups, threads, 0, stream>>>(logits, pitch, chosen, mask, tokens, experts, choices, g.per,
                                                                               coefficient, out, sums, counts, counted, finished);
  });
  if (g.groups > 1)
    finish_forward<><<<finish_groups(experts), threads, 0, stream>>>(sums, counts, counted, g.groups, experts, choices, coefficient, out, parts, finished);
  return static_cast<int>(hipGetLastError());
}

template <typename type_t>
int launch_backward(hipStream_t stream, const type_t* logits, std::size_t pitch, const int* counts, const int* counted, const unsigned char* mask,
                    int tokens, int experts, int choices, float coefficient, const float* grad_loss, type_t* grad, std::size_t grad_pitch) {
  if (tokens == 0) return 0;
  with_shape<type_t>(experts, [&](auto full, auto v, auto lanes, auto k) {
    constexpr bool FULL = decltype(full)::value;
    constexpr int V = decltype(v)::value, G = decltype(lanes)::value, K = decltype(k)::value, U = K == 1 ? 2 : 1;
    constexpr int rows = 4 * (wave::size / G);
    const long long groups = (static_cast<long long>(tokens) + rows - 1) / rows;
    const unsigned int grid = static_cast<unsigned int>(groups < 8192 ? groups : 8192);
    backward<FULL, V, G, K, U, type_t><<<grid, 256, 0, stream>>>(logits, pitch, counts, counted, mask, tokens, experts, choices, coefficient, grad_loss, grad,
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
