// Log probabilities of given tokens, with the entropy of each row's
// distribution and its most likely alternatives, and their gradient.
#include <torch/csrc/utils/pybind.h>

#include "token_losses.cuh"

namespace kb {
namespace {

constexpr int kCand = 2048;  // candidates held while the alternatives are selected
constexpr int kStats = 2;    // floats kept per row for the backward pass: m, log2 S

// ----------------------------------------------------------- alternatives

// Order of floats as unsigned integers: NaN above +inf, the two zeros equal, -inf above 0 (no element).
__device__ __forceinline__ uint32_t order_of(float v) {
  if (v != v) return 0xFFFFFFFFu;
  const uint32_t b = __float_as_uint(v + 0.f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t o) {
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7FFFFFFFu) : ~o);
}
// Larger value first, then the lower index; all keys of a row differ.
__device__ __forceinline__ unsigned long long key_of(uint32_t order, int index) {
  return ((unsigned long long)order << 32) | (uint32_t)~index;
}

struct SelectShared {
  unsigned long long cand[kCand];
  unsigned long long sorted[kMaxList];
  uint32_t wmin[32], wmax[32];
  int count, listed;
  int warp_sum[32];
  uint16_t tids[1024];
};

// The k largest keys of a block's elements, sorted, in sh.sorted (padded with
// 0 where the block has fewer).
//
// Selection without a second pass over the row: every thread knows the
// maximum of its own elements. If t is the k-th largest of the thread maxima,
// at least k elements are >= t, so only the threads whose maximum is >= t
// (about k of them) hold elements of the answer. t is found by bisection on
// the integer order, one vote of the block per step; it may stop early at a
// slightly lower t. The elements of those threads are read again (from L2)
// by the whole block and those >= t are ranked by counting.
// Ties and rows sorted in memory can make the candidates overflow; then the
// k-th value is bisected over the row itself and ties are taken in index order.
template <typename T, int NT>
__device__ void select_top(const Row<T>& row, int u0, int u1, int ragged, float mine, int k, SelectShared& sh) {
  constexpr int E = Elem<T>::kUnit;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n_units = u1 - u0;
  const int total = n_units * E + ragged;
  const int want = min(k, total);
  const bool has = tid < n_units || tid < ragged;
  const uint32_t key = has ? order_of(mine) : 0u;
  const uint32_t wmin = __reduce_min_sync(0xffffffffu, key), wmax = __reduce_max_sync(0xffffffffu, key);
  if (lane == 0) {
    sh.wmin[warp] = wmin;
    sh.wmax[warp] = wmax;
  }
  if (tid == 0) {
    sh.count = 0;
    sh.listed = 0;
  }
  for (int i = tid; i < k; i += NT) sh.sorted[i] = 0;
  __syncthreads();
  uint32_t lo = 0xFFFFFFFFu, top = 0u;
  for (int w = 0; w < NT / 32; ++w) {
    lo = min(lo, sh.wmin[w]);
    top = max(top, sh.wmax[w]);
  }
  // count(key >= lo) >= want, count(key > hi) < want; with fewer threads than `want` every element stays.
  if (want > NT) lo = 0;
  uint32_t hi = want > NT ? 0u : top;
  const int enough = want + (want >> 2) + 4;
  while (lo < hi) {
    const uint32_t mid = lo + (hi - lo) / 2 + 1;
    const int n = __syncthreads_count(key >= mid);
    if (n >= want) {
      lo = mid;
      if (n <= enough) break;
    } else {
      hi = mid - 1;
    }
  }
  const uint32_t t = max(lo, 1u);
  if (key >= t) sh.tids[atomicAdd(&sh.listed, 1)] = (uint16_t)tid;
  __syncthreads();
  const int per = (n_units + NT - 1) / NT + 1;  // a thread's units, and one ragged element
  const int tasks = sh.listed * per;
  const uint4* p = row.unit_ptr();
  for (int i = tid; i < tasks; i += NT) {
    const int who = sh.tids[i / per], j = i % per;
    if (j == per - 1) {
      if (who < ragged) {
        const int idx = row.ragged_index(who);
        const uint32_t o = order_of(Elem<T>::load(row.z + idx));
        if (o >= t) {
          const int at = atomicAdd(&sh.count, 1);
          if (at < kCand) sh.cand[at] = key_of(o, idx);
        }
      }
    } else {
      const int u = u0 + who + j * NT;
      if (u < u1) {
        const uint4 q = load_unit(p + u);
        float v[E];
        Elem<T>::unpack(q, v);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const uint32_t o = order_of(v[e]);
          if (o >= t) {
            const int at = atomicAdd(&sh.count, 1);
            if (at < kCand) sh.cand[at] = key_of(o, row.head + u * E + e);
          }
        }
      }
    }
  }
  __syncthreads();
  int n = sh.count;
  __syncthreads();
  if (n > kCand) {
    // The want-th value over all elements: count(>= lo) >= want and count(> hi) < want throughout.
    auto count_from = [&](uint32_t bound) {
      if (tid == 0) sh.count = 0;
      __syncthreads();
      int mine_n = 0;
      for (int u = u0 + tid; u < u1; u += NT) {
        float v[E];
        Elem<T>::unpack(load_unit(p + u), v);
#pragma unroll
        for (int e = 0; e < E; ++e) mine_n += order_of(v[e]) >= bound;
      }
      if (tid < ragged) mine_n += order_of(Elem<T>::load(row.z + row.ragged_index(tid))) >= bound;
      mine_n = __reduce_add_sync(0xffffffffu, mine_n);
      if (lane == 0) atomicAdd(&sh.count, mine_n);
      __syncthreads();
      const int r = sh.count;
      __syncthreads();
      return r;
    };
    uint32_t a = t, b = top;
    bool first = true;
    while (a < b) {
      const uint32_t mid = first ? a + 1 : a + (b - a) / 2 + 1;  // most often t itself is the value
      first = false;
      if (count_from(mid) >= want) a = mid;
      else b = mid - 1;
    }
    if (tid == 0) sh.count = 0;
    __syncthreads();
    // All elements above it, fewer than `want`; then the ties in index order.
    auto take_above = [&](uint32_t o, int idx) {
      if (o > a) sh.cand[atomicAdd(&sh.count, 1)] = key_of(o, idx);
    };
    for (int u = u0 + tid; u < u1; u += NT) {
      float v[E];
      Elem<T>::unpack(load_unit(p + u), v);
#pragma unroll
      for (int e = 0; e < E; ++e) take_above(order_of(v[e]), row.head + u * E + e);
    }
    if (tid < ragged) take_above(order_of(Elem<T>::load(row.z + row.ragged_index(tid))), row.ragged_index(tid));
    __syncthreads();
    int taken = sh.count;
    // Index order: the head's ragged elements, the units, the tail's; a block without ragged elements has units only.
    const int first_idx = ragged ? 0 : row.head + u0 * E;
    const int unit_end = row.head + u1 * E;
    const int tail = ragged ? row.head + row.units * E : unit_end, end = ragged ? ragged + row.units * E : unit_end;
    for (int base = first_idx; base < end && taken < want; base += NT) {
      const int idx = base + tid;
      const bool in = idx < unit_end || (idx >= tail && idx < end);
      const bool tie = in && order_of(Elem<T>::load(row.z + idx)) == a;
      const uint32_t vote = __ballot_sync(0xffffffffu, tie);
      if (lane == 0) sh.warp_sum[warp] = __popc(vote);
      __syncthreads();
      int before = taken, sum = 0;
      for (int w = 0; w < NT / 32; ++w) {
        if (w < warp) before += sh.warp_sum[w];
        sum += sh.warp_sum[w];
      }
      const int at = before + __popc(vote & ((1u << lane) - 1u));
      if (tie && at < want) sh.cand[at] = key_of(a, idx);
      taken = min(want, taken + sum);
      __syncthreads();
    }
    n = want;
  } else if (n > 2 * want + 64) {
    // Too many to rank by counting: cut by a bisected key first.
    unsigned long long klo = 0, khi = ~0ull;
    while (klo < khi) {
      const unsigned long long mid = klo + (khi - klo) / 2 + 1;
      int got = 0;
      for (int i = 0; i < n; i += NT) got += __syncthreads_count(i + tid < n && sh.cand[i + tid] >= mid);
      if (got >= want) {
        klo = mid;
        if (got <= 2 * want + 64) break;
      } else {
        khi = mid - 1;
      }
    }
    constexpr int PER = kCand / NT;
    unsigned long long keep[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) keep[i] = i * NT + tid < n ? sh.cand[i * NT + tid] : 0ull;
    if (tid == 0) sh.count = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (keep[i] != 0 && keep[i] >= klo) sh.cand[atomicAdd(&sh.count, 1)] = keep[i];
    __syncthreads();
    n = sh.count;
  }
  for (int i = tid; i < n; i += NT) {
    const unsigned long long ki = sh.cand[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += sh.cand[j] > ki;
    if (rank < want) sh.sorted[rank] = ki;
  }
  __syncthreads();
}

// --------------------------------------------------- log probabilities

// One block per row: statistics in one pass, then the alternatives.
template <typename T, int NT, bool TOPK>
__global__ void __launch_bounds__(NT) logprob_forward_kernel(const T* __restrict__ logits, long long ld, int V,
                                                             const int64_t* __restrict__ tokens, int64_t ignore_index,
                                                             float c, float inv_t, int k, float* __restrict__ logprobs,
                                                             float* __restrict__ entropy, float* __restrict__ stats,
                                                             float* __restrict__ top_logprobs,
                                                             int64_t* __restrict__ top_ids) {
  const int row_i = blockIdx.x, tid = threadIdx.x;
  const int64_t token = tokens ? tokens[row_i] : 0;
  if (tokens && token == ignore_index) {
    if (tid == 0) {
      logprobs[row_i] = 0.f;
      entropy[row_i] = 0.f;
      stats[kStats * (long long)row_i] = 0.f;
      stats[kStats * (long long)row_i + 1] = 0.f;
    }
    if (TOPK) {
      for (int i = tid; i < k; i += NT) {
        top_logprobs[(long long)row_i * k + i] = 0.f;
        top_ids[(long long)row_i * k + i] = -1;
      }
    }
    return;
  }
  const Row<T> row(logits + (long long)row_i * ld, V);
  Acc acc;
  if (tid < row.ragged) {
    const float v = Elem<T>::load(row.z + row.ragged_index(tid));
    const float ms = acc.raise<true>(v, c);
    acc.add<true>(v, ms, c);
  }
  stream_units<T, NT, true, false>(row.unit_ptr(), 0, row.units, c, acc, nullptr);
  __shared__ float join_sm[32][3];
  const Acc all = block_join<NT, true>(acc, c, join_sm);
  // Log probabilities are taken in units of z / T, not of c z: (lowest - m) c would overflow.
  const float log2s = log2f(all.s), ln_s = kLn2 * log2s;
  if (tid == 0) {
    if (tokens) {
      const bool inside = token >= 0 && token < V;
      logprobs[row_i] = inside ? (Elem<T>::load(row.z + token) - all.m) * inv_t - ln_s : NAN;
    }
    entropy[row_i] = kLn2 * (log2s - all.a / all.s);
    stats[kStats * (long long)row_i] = all.m;
    stats[kStats * (long long)row_i + 1] = log2s;
  }
  if constexpr (TOPK) {
    __shared__ SelectShared sh;
    select_top<T, NT>(row, 0, row.units, row.ragged, acc.m, k, sh);
    for (int i = tid; i < k; i += NT) {
      const unsigned long long key = sh.sorted[i];
      top_ids[(long long)row_i * k + i] = (int64_t)(uint32_t)~(uint32_t)key;
      top_logprobs[(long long)row_i * k + i] = (value_of((uint32_t)(key >> 32)) - all.m) * inv_t - ln_s;
    }
  }
}

// dz_j = 1/T [ dlp (1[j = token] - p_j) - dH p_j (ln p_j + H) ], p_j = 2^y_j with y_j = (z_j - m) c - log2 S.
// One pass, rows cut into gridDim.y segments.
template <typename T, int NT>
__global__ void __launch_bounds__(NT)
    logprob_backward_kernel(const T* logits, long long ld, T* out, long long ld_out, int V,
                            const int64_t* __restrict__ tokens, int64_t ignore_index, float c, float inv_t,
                            const float* __restrict__ stats, const float* __restrict__ entropy,
                            const float* __restrict__ dlogprobs, const float* __restrict__ dentropy) {
  const int row_i = blockIdx.x;
  const int64_t token = tokens ? tokens[row_i] : -1;
  float g = dlogprobs ? dlogprobs[row_i] : 0.f;
  const float gh = dentropy ? dentropy[row_i] : 0.f;
  int u0, u1;
  if ((tokens && token == ignore_index) || (g == 0.f && gh == 0.f)) {
    const Row<T> row(out + (long long)row_i * ld_out, V);
    segment(row.units, blockIdx.y, gridDim.y, u0, u1);
    zero_row<T, NT>(row, u0, u1, blockIdx.y == 0 ? row.ragged : 0);
    return;
  }
  if (token < 0 || token >= V) g = g == 0.f ? 0.f : NAN;  // its log probability is NaN too
  const Row<T> row(logits + (long long)row_i * ld, V);
  segment(row.units, blockIdx.y, gridDim.y, u0, u1);
  const float m = stats[kStats * (long long)row_i], log2s = stats[kStats * (long long)row_i + 1];
  const float a = -(g + gh * entropy[row_i]) * inv_t, b = -gh * kLn2 * inv_t, hot = g * inv_t;
  const int at = (int)token;
  map_row<T, NT>(row, out + (long long)row_i * ld_out, u0, u1, blockIdx.y == 0 ? row.ragged : 0, [&](float z, int j) {
    const float y = (z - m) * c - log2s;
    const float d = ex2(y) * fmaf(b, fmaxf(y, -256.f), a);
    return j == at ? d + hot : d;
  });
}

}  // namespace

void token_logprobs_forward(const at::Tensor& logits, const c10::optional<at::Tensor>& tokens,
                            const c10::optional<at::Tensor>& logprobs, at::Tensor& entropy, at::Tensor& stats,
                            const c10::optional<at::Tensor>& top_logprobs, const c10::optional<at::Tensor>& top_ids,
                            int64_t vocab, double temperature, int64_t ignore_index) {
  const int64_t rows = check_logits(logits, vocab, temperature, "logits");
  KB_CHECK(tokens.has_value() == logprobs.has_value(), "tokens and logprobs go together");
  KB_CHECK(top_logprobs.has_value() == top_ids.has_value(), "top_logprobs and top_ids go together");
  if (tokens) check_rows(*tokens, "tokens", rows, 1, at::kLong, logits);
  if (logprobs) check_rows(*logprobs, "logprobs", rows, 1, at::kFloat, logits);
  check_rows(entropy, "entropy", rows, 1, at::kFloat, logits);
  check_rows(stats, "stats", rows, kStats, at::kFloat, logits);
  int k = 0;
  if (top_ids) {
    KB_CHECK(top_ids->dim() == 2, "top_ids must be [rows, k]");
    KB_CHECK(top_ids->size(1) >= 1 && top_ids->size(1) <= std::min<int64_t>(kMaxList, vocab),
             "1 to 128 alternatives, and no more than the vocabulary holds");
    k = (int)top_ids->size(1);
    check_rows(*top_ids, "top_ids", rows, k, at::kLong, logits);
    check_rows(*top_logprobs, "top_logprobs", rows, k, at::kFloat, logits);
  }
  if (rows == 0) return;
  const c10::cuda::CUDAGuard guard(logits.device());
  cudaStream_t s = c10::cuda::getCurrentCUDAStream().stream();
  const float c = (float)(1.4426950408889634 / temperature);
  const int64_t* tok = tokens ? tokens->data_ptr<int64_t>() : nullptr;
  float* lp = logprobs ? logprobs->data_ptr<float>() : nullptr;
  float* tl = top_logprobs ? top_logprobs->data_ptr<float>() : nullptr;
  int64_t* ti = top_ids ? top_ids->data_ptr<int64_t>() : nullptr;
  for_logits_type(logits.scalar_type(), [&](auto tag) {
    using T = typename decltype(tag)::type;
    auto launch = [&](auto kern, int nt) {
      kern<<<(unsigned)rows, nt, 0, s>>>((const T*)logits.data_ptr(), logits.stride(0), (int)vocab, tok, ignore_index,
                                         c, (float)(1.0 / temperature), k, lp, entropy.data_ptr<float>(), stats.data_ptr<float>(), tl, ti);
    };
    const bool small = vocab * (int64_t)sizeof(T) <= 8192;
    if (small) k ? launch(logprob_forward_kernel<T, 128, true>, 128) : launch(logprob_forward_kernel<T, 128, false>, 128);
    else k ? launch(logprob_forward_kernel<T, 512, true>, 512) : launch(logprob_forward_kernel<T, 512, false>, 512);
  });
  KB_LAUNCHED();
}

void token_logprobs_backward(const at::Tensor& logits, const c10::optional<at::Tensor>& tokens,
                             const at::Tensor& stats, const at::Tensor& entropy,
                             const c10::optional<at::Tensor>& dlogprobs, const c10::optional<at::Tensor>& dentropy,
                             at::Tensor& out, int64_t vocab, double temperature, int64_t ignore_index) {
  const int64_t rows = check_logits(logits, vocab, temperature, "logits");
  check_out(out, logits, vocab);
  if (tokens) check_rows(*tokens, "tokens", rows, 1, at::kLong, logits);
  KB_CHECK(tokens.has_value() || !dlogprobs.has_value(), "dlogprobs without tokens");
  check_rows(stats, "stats", rows, kStats, at::kFloat, logits);
  check_rows(entropy, "entropy", rows, 1, at::kFloat, logits);
  if (dlogprobs) check_rows(*dlogprobs, "dlogprobs", rows, 1, at::kFloat, logits);
  if (dentropy) check_rows(*dentropy, "dentropy", rows, 1, at::kFloat, logits);
  if (rows == 0) return;
  const c10::cuda::CUDAGuard guard(logits.device());
  cudaStream_t s = c10::cuda::getCurrentCUDAStream().stream();
  const float c = (float)(1.4426950408889634 / temperature);
  for_logits_type(logits.scalar_type(), [&](auto tag) {
    using T = typename decltype(tag)::type;
    const int nseg = row_segments(rows, vocab, sizeof(T), 256, logits.get_device());
    logprob_backward_kernel<T, 256><<<dim3((unsigned)rows, nseg), 256, 0, s>>>(
        (const T*)logits.data_ptr(), logits.stride(0), (T*)out.data_ptr(), out.stride(0), (int)vocab,
        tokens ? tokens->data_ptr<int64_t>() : nullptr, ignore_index, c, (float)(1.0 / temperature),
        stats.data_ptr<float>(), entropy.data_ptr<float>(), dlogprobs ? dlogprobs->data_ptr<float>() : nullptr,
        dentropy ? dentropy->data_ptr<float>() : nullptr);
  });
  KB_LAUNCHED();
}

void register_token_logprobs_ops(pybind11::module& m) {
  m.def("token_logprobs_forward", &token_logprobs_forward,
        "log probabilities of given tokens, entropies and the most likely alternatives");
  m.def("token_logprobs_backward", &token_logprobs_backward, "gradient of log probabilities and entropies");
  m.attr("TOKEN_LOGPROBS_STATS") = kStats;
}

}  // namespace kb
