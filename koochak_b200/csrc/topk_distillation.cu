// Distillation from a teacher known by its top logits: KL divergence of the
// student's distribution from the teacher's, and its gradient.
#include <torch/csrc/utils/pybind.h>

#include "token_losses.cuh"

namespace kb {
namespace {

constexpr int kStats = 8;  // floats kept per row for the backward pass: KdStats, the last 0 for a row without slots

// --------------------------------------------------------- distillation

struct ListShared {
  int id[kMaxList];
  float t[kMaxList], z[kMaxList], q[kMaxList];
  int repeated;
};

// Reads a row's slots: ids (-1 where empty), teacher values and the student's logits there. Returns whether any is
// valid.
template <typename T, int NT>
__device__ __forceinline__ bool read_slots(const T* z, int V, const int64_t* ids, const float* teacher, int K,
                                           ListShared& sh) {
  bool any = false;
  for (int i = threadIdx.x; i < K; i += NT) {
    const int64_t id = ids[i];
    const bool ok = id >= 0 && id < V;
    sh.id[i] = ok ? (int)id : -1;
    sh.t[i] = ok ? teacher[i] : -INFINITY;
    sh.z[i] = ok ? Elem<T>::load(z + id) : 0.f;
    any |= ok;
  }
  return __syncthreads_or(any);
}

// What a row's gradient needs besides its logits:
// dz_j = g (coef 2^((z_j - ms) c)) off the list, g (Q p_j - sum of its q) on it, p_j = 2^((z_j - m) c) inv_s.
struct KdStats {
  float ms, coef, m, inv_s, t_max, inv_e, mass, loss;
};

// Loss of one row, by one warp, from the statistics of the streamed elements
// (all of them, or with TAIL those off the list).
template <bool TAIL>
__device__ __forceinline__ KdStats distill_row(const Acc& str, float c, float inv_t, int K, const ListShared& sh) {
  const int lane = threadIdx.x & 31;
  KdStats r;
  float q_sum = 0.f;
  if (TAIL) {
    r.t_max = 0.f;
    r.inv_e = 1.f;
    for (int i = lane; i < K; i += 32) q_sum += ex2(sh.t[i] * kLog2e);
    q_sum = warp_sum(q_sum);
  } else {
    float tm = -INFINITY, e = 0.f;
    for (int i = lane; i < K; i += 32) tm = max_nan(tm, sh.t[i]);
    tm = warp_max_nan(tm);
    r.t_max = tm == -INFINITY ? 0.f : tm;
    for (int i = lane; i < K; i += 32) e += ex2((sh.t[i] - r.t_max) * c);
    e = warp_sum(e);
    r.inv_e = e == 0.f ? 0.f : 1.f / e;
    q_sum = e == 0.f ? 0.f : 1.f;
  }
  const float q_rest = TAIL ? (q_sum > 1.f ? 0.f : 1.f - q_sum) : 0.f;
  Acc all = str;
  if (TAIL) {
    float zm = -INFINITY;
    for (int i = lane; i < K; i += 32)
      if (sh.id[i] >= 0) zm = max_nan(zm, sh.z[i]);
    zm = warp_max_nan(zm);
    const float zs = zm == -INFINITY ? 0.f : zm;
    float s = 0.f;
    for (int i = lane; i < K; i += 32) {
      bool counts = sh.id[i] >= 0;
      if (sh.repeated)
        for (int j = 0; j < i; ++j) counts &= sh.id[j] != sh.id[i];
      if (counts) s += ex2((sh.z[i] - zs) * c);
    }
    s = warp_sum(s);
    all.join<false>(zm, s, 0.f, c);
  }
  // In units of z / T, not of c z: (lowest - m) c would overflow.
  const float ln_s = kLn2 * log2f(all.s), ln_inv_e = TAIL ? 0.f : kLn2 * log2f(r.inv_e);
  float loss = 0.f;
  for (int i = lane; i < K; i += 32) {
    const float t = sh.t[i] - r.t_max;
    const float q = ex2(t * (TAIL ? kLog2e : c)) * r.inv_e;
    const float lq = TAIL ? t : t * inv_t + ln_inv_e;
    if (q != 0.f) loss += q * (lq - ((sh.z[i] - all.m) * inv_t - ln_s));
  }
  loss = warp_sum(loss);
  r.m = all.m;
  r.inv_s = 1.f / all.s;
  // Where the student has no mass off the list, a rest is an infinite constant: it has no gradient.
  r.mass = TAIL && str.s != 0.f ? q_sum + q_rest : q_sum;
  if (TAIL) {
    const float down = str.m == all.m ? 0.f : str.m - all.m;
    if (q_rest != 0.f) loss += q_rest * (kLn2 * (log2f(q_rest) - log2f(str.s)) - down * inv_t + ln_s);
    r.coef = str.s == 0.f ? 0.f : r.mass * ex2(down * c) * r.inv_s - q_rest / str.s;
  } else {
    r.coef = r.mass * r.inv_s;
  }
  r.ms = str.m == -INFINITY ? 0.f : str.m;
  r.loss = loss;
  return r;
}

// One block per row. Off-list elements are told by a bit per element in shared memory (TAIL).
template <typename T, int NT, bool TAIL>
__global__ void __launch_bounds__(NT)
    distill_forward_kernel(const T* __restrict__ logits, long long ld, int V, const int64_t* __restrict__ ids,
                           const float* __restrict__ teacher, int K, float c, float inv_t, float* __restrict__ loss,
                           float* __restrict__ stats) {
  extern __shared__ __align__(16) uint8_t bits[];
  __shared__ ListShared sh;
  __shared__ Acc join_sm[NT / 32];
  constexpr int E = Elem<T>::kUnit;
  const int tid = threadIdx.x;
  const long long row_i = blockIdx.x;
  const Row<T> row(logits + row_i * ld, V);
  if (tid == 0) sh.repeated = 0;
  if (TAIL) {
    uint32_t* w = reinterpret_cast<uint32_t*>(bits);
    for (int i = tid; i < (V + 31) / 32; i += NT) w[i] = 0;
  }
  if (!read_slots<T, NT>(row.z, V, ids + row_i * K, teacher + row_i * K, K, sh)) {
    if (tid == 0) loss[row_i] = 0.f;
    if (tid < kStats) stats[row_i * kStats + tid] = 0.f;
    return;
  }
  Run<false> run;
  if (TAIL) {
    // Bit u * E + j for element j of unit u, ragged elements behind the units.
    for (int i = tid; i < K; i += NT) {
      const int id = sh.id[i];
      if (id < 0) continue;
      const int body = row.units * E;
      const int bit = id < row.head ? body + id : id < row.head + body ? id - row.head : id;
      const uint32_t old = atomicOr(reinterpret_cast<uint32_t*>(bits) + (bit >> 5), 1u << (bit & 31));
      if ((old >> (bit & 31)) & 1u) sh.repeated = 1;
    }
    __syncthreads();
  }
  if (tid < 32) {  // fewer than two units of ragged elements
    const int bit = row.units * E + tid;
    const bool in = tid < row.ragged && (!TAIL || !((bits[bit >> 3] >> (bit & 7)) & 1u));
    run.add_one(in ? Elem<T>::load(row.z + row.ragged_index(tid)) : -INFINITY, c);
  }
  stream_units<T, NT, false, TAIL>(row.unit_ptr(), 0, row.units, c, run, bits, [](int, float) {});
  const Acc all = block_join<NT, false>(run, c, join_sm);
  if (tid < 32) {
    const KdStats r = distill_row<TAIL>(all, c, inv_t, K, sh);
    if (tid == 0) {
      loss[row_i] = r.loss;
      float* s = stats + row_i * kStats;
      s[0] = r.ms;
      s[1] = r.coef;
      s[2] = r.m;
      s[3] = r.inv_s;
      s[4] = r.t_max;
      s[5] = r.inv_e;
      s[6] = r.mass;
      s[7] = 1.f;
    }
  }
}

// Gradient of the listed elements of a segment: sums the q of slots that name the same token.
template <typename T, int NT, bool TAIL>
__device__ __forceinline__ void write_listed(T* out, const ListShared& sh, int K, float c, float g, const KdStats& r,
                                             int lo, int hi, bool ragged_too, int body_lo, int body_hi) {
  for (int i = threadIdx.x; i < K; i += NT) {
    const int id = sh.id[i];
    if (id < 0) continue;
    const bool in_body = id >= body_lo && id < body_hi;
    if (in_body ? !(id >= lo && id < hi) : !ragged_too) continue;
    float q = 0.f;
    for (int j = 0; j < K; ++j)
      if (sh.id[j] == id) q += sh.q[j];
    Elem<T>::store(out + id, g * (r.mass * (ex2((sh.z[i] - r.m) * c) * r.inv_s) - q));
  }
}

template <typename T, int NT, bool TAIL>
__global__ void __launch_bounds__(NT)
    distill_backward_kernel(const T* logits, long long ld, T* out, long long ld_out, int V,
                            const int64_t* __restrict__ ids, const float* __restrict__ teacher, int K, float c,
                            float inv_t, const float* __restrict__ stats, const float* __restrict__ row_scale,
                            const float* __restrict__ scale) {
  constexpr int E = Elem<T>::kUnit;
  __shared__ ListShared sh;
  const long long row_i = gridDim.x - 1 - blockIdx.x;  // last rows first: the forward pass left them in L2
  const float* s = stats + row_i * kStats;
  const float w = row_scale ? row_scale[row_i] : 1.f;
  T* o = out + row_i * ld_out;
  int u0, u1;
  if (s[7] == 0.f || w == 0.f) {
    const Row<T> row(o, V);
    segment(row.units, blockIdx.y, gridDim.y, u0, u1);
    zero_row<T, NT>(row, u0, u1, blockIdx.y == 0 ? row.ragged : 0);
    return;
  }
  const Row<T> row(logits + row_i * ld, V);
  segment(row.units, blockIdx.y, gridDim.y, u0, u1);
  KdStats r;
  r.ms = s[0];
  r.coef = s[1];
  r.m = s[2];
  r.inv_s = s[3];
  r.t_max = s[4];
  r.inv_e = s[5];
  r.mass = s[6];
  const float g = w * (scale ? *scale : 1.f) * inv_t;
  read_slots<T, NT>(row.z, V, ids + row_i * K, teacher + row_i * K, K, sh);
  for (int i = threadIdx.x; i < K; i += NT) sh.q[i] = ex2((sh.t[i] - r.t_max) * (TAIL ? kLog2e : c)) * r.inv_e;
  const float dense = g * r.coef;
  const int ragged = blockIdx.y == 0 ? row.ragged : 0;
  const F2 minus_m = pair(-r.ms, -r.ms), cc = pair(c, c), dd = pair(dense, dense);
  map_row<T, NT>(row, o, u0, u1, ragged, [&](F2 z, int) {
    const float2 x = split(mul2(add2(z, minus_m), cc));
    return mul2(pair(ex2(x.x), ex2(x.y)), dd);
  });
  __syncthreads();
  write_listed<T, NT, TAIL>(o, sh, K, c, g, r, row.head + u0 * E, row.head + u1 * E, blockIdx.y == 0, row.head,
                            row.head + row.units * E);
}

int check_teacher(const at::Tensor& ids, const at::Tensor& teacher, int64_t rows, const at::Tensor& logits) {
  KB_CHECK(ids.dim() == 2 && ids.size(1) >= 1 && ids.size(1) <= kMaxList, "1 to 128 teacher slots per row");
  const int k = (int)ids.size(1);
  check_rows(ids, "teacher_ids", rows, k, at::kLong, logits);
  check_rows(teacher, "teacher_logits", rows, k, at::kFloat, logits);
  return k;
}
}  // namespace

void topk_distillation_forward(const at::Tensor& logits, const at::Tensor& ids, const at::Tensor& teacher,
                               at::Tensor& loss, at::Tensor& stats, int64_t vocab, double temperature, bool tail) {
  const int64_t rows = check_logits(logits, vocab, temperature, "logits");
  const int k = check_teacher(ids, teacher, rows, logits);
  check_rows(loss, "loss", rows, 1, at::kFloat, logits);
  check_rows(stats, "stats", rows, kStats, at::kFloat, logits);
  if (rows == 0) return;
  const c10::cuda::CUDAGuard guard(logits.device());
  cudaStream_t s = c10::cuda::getCurrentCUDAStream().stream();
  const float c = (float)(1.4426950408889634 / temperature);
  const size_t bits = tail ? (size_t)((vocab + 31) / 32 * 4) : 0;
  for_logits_type(logits.scalar_type(), [&](auto tag) {
    using T = typename decltype(tag)::type;
    auto launch = [&](auto kern, int nt) {
      if (bits > 32 * 1024)
        KB_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bits));
      kern<<<(unsigned)rows, nt, bits, s>>>((const T*)logits.data_ptr(), logits.stride(0), (int)vocab,
                                            ids.data_ptr<int64_t>(), teacher.data_ptr<float>(), k, c,
                                            (float)(1.0 / temperature), loss.data_ptr<float>(), stats.data_ptr<float>());
    };
    const int nt = getenv("KB_NT") ? atoi(getenv("KB_NT")) : 512;
    if (nt == 128) tail ? launch(distill_forward_kernel<T, 128, true>, 128) : launch(distill_forward_kernel<T, 128, false>, 128);
    else if (nt == 256) tail ? launch(distill_forward_kernel<T, 256, true>, 256) : launch(distill_forward_kernel<T, 256, false>, 256);
    else tail ? launch(distill_forward_kernel<T, 512, true>, 512) : launch(distill_forward_kernel<T, 512, false>, 512);
  });
  KB_LAUNCHED();
}

void topk_distillation_backward(const at::Tensor& logits, const at::Tensor& ids, const at::Tensor& teacher,
                                const at::Tensor& stats, const c10::optional<at::Tensor>& row_scale,
                                const c10::optional<at::Tensor>& scale, at::Tensor& out, int64_t vocab,
                                double temperature, bool tail) {
  const int64_t rows = check_logits(logits, vocab, temperature, "logits");
  check_out(out, logits, vocab);
  const int k = check_teacher(ids, teacher, rows, logits);
  check_rows(stats, "stats", rows, kStats, at::kFloat, logits);
  if (row_scale) check_rows(*row_scale, "row_scale", rows, 1, at::kFloat, logits);
  if (scale) check_rows(*scale, "scale", 1, 1, at::kFloat, logits);
  if (rows == 0) return;
  const c10::cuda::CUDAGuard guard(logits.device());
  cudaStream_t s = c10::cuda::getCurrentCUDAStream().stream();
  const float c = (float)(1.4426950408889634 / temperature);
  for_logits_type(logits.scalar_type(), [&](auto tag) {
    using T = typename decltype(tag)::type;
    const int nseg = row_segments(rows, vocab, sizeof(T), 256, logits.get_device());
    auto launch = [&](auto kern) {
      kern<<<dim3((unsigned)rows, nseg), 256, 0, s>>>(
          (const T*)logits.data_ptr(), logits.stride(0), (T*)out.data_ptr(), out.stride(0), (int)vocab,
          ids.data_ptr<int64_t>(), teacher.data_ptr<float>(), k, c, (float)(1.0 / temperature),
          stats.data_ptr<float>(), row_scale ? row_scale->data_ptr<float>() : nullptr,
          scale ? scale->data_ptr<float>() : nullptr);
    };
    tail ? launch(distill_backward_kernel<T, 256, true>) : launch(distill_backward_kernel<T, 256, false>);
  });
  KB_LAUNCHED();
}

void register_topk_distillation_ops(pybind11::module& m) {
  m.def("topk_distillation_forward", &topk_distillation_forward, "KL divergence from a teacher's top logits");
  m.def("topk_distillation_backward", &topk_distillation_backward, "gradient of topk_distillation_forward");
  m.attr("TOPK_DISTILLATION_STATS") = kStats;
}

}  // namespace kb
