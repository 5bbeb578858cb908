// Distillation from a teacher known by its top logits: KL divergence of the
// student's distribution from the teacher's, and its gradient.
#include <torch/csrc/utils/pybind.h>

#include "sm100.cuh"
#include "token_losses.cuh"

namespace kb {
namespace {

constexpr int kGradThreads = 512;  // streaming threads of the kernel that writes loss and gradient
constexpr int kStageBytes = 107 * 1024;  // of staged units and marks, for two blocks on an SM
constexpr int kChunks = (kStageBytes / 16 + kBatch * kGradThreads - 1) / (kBatch * kGradThreads);  // bulk copies of a row
constexpr int kStats = kTopkDistillationStats;  // KdStats, and 0 for a row without slots

// --------------------------------------------------------- distillation

struct ListShared {
  int id[kMaxList];
  float t[kMaxList], z[kMaxList], q[kMaxList];
  int repeated;
};

// Reads a row's slots: ids (-1 where empty), teacher values and the student's logits there. Returns whether the
// thread's are any valid.
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
  return any;
}

// What a row's gradient needs besides its logits:
// dz_j = g (coef 2^((z_j - ms) c)) off the list, g (Q p_j - sum of its q) on it, p_j = 2^((z_j - m) c) inv_s.
struct KdStats {
  float ms, coef, m, inv_s, t_max, inv_e, mass;
};
__device__ __forceinline__ void store_stats(float* s, const KdStats& r) {
  s[0] = r.ms;
  s[1] = r.coef;
  s[2] = r.m;
  s[3] = r.inv_s;
  s[4] = r.t_max;
  s[5] = r.inv_e;
  s[6] = r.mass;
  s[7] = 1.f;
}

// What a row's list alone decides: the normaliser of q, its sum, the rest, and (TAIL) the student's maximum and sum
// over the distinct listed tokens.
struct ListStats {
  float t_max, inv_e, q_sum, q_rest, z_max, z_sum;
};

// By one warp.
template <bool TAIL>
__device__ __forceinline__ ListStats list_stats(float c, int K, const ListShared& sh) {
  const int lane = threadIdx.x & 31;
  ListStats r{0.f, 1.f, 0.f, 0.f, -INFINITY, 0.f};
  if (TAIL) {
    float q_sum = 0.f, zm = -INFINITY, s = 0.f;
    for (int i = lane; i < K; i += 32) {
      q_sum += ex2(sh.t[i] * kLog2e);
      if (sh.id[i] >= 0) zm = max_nan(zm, sh.z[i]);
    }
    r.q_sum = warp_sum(q_sum);
    r.q_rest = r.q_sum > 1.f ? 0.f : 1.f - r.q_sum;
    r.z_max = warp_max_nan(zm);
    const float zs = r.z_max == -INFINITY ? 0.f : r.z_max;
    for (int i = lane; i < K; i += 32) {
      bool counts = sh.id[i] >= 0;
      if (sh.repeated)
        for (int j = 0; j < i; ++j) counts &= sh.id[j] != sh.id[i];
      if (counts) s += ex2((sh.z[i] - zs) * c);
    }
    r.z_sum = warp_sum(s);
  } else {
    float tm = -INFINITY, e = 0.f;
    for (int i = lane; i < K; i += 32) tm = max_nan(tm, sh.t[i]);
    tm = warp_max_nan(tm);
    r.t_max = tm == -INFINITY ? 0.f : tm;
    for (int i = lane; i < K; i += 32) e += ex2((sh.t[i] - r.t_max) * c);
    e = warp_sum(e);
    r.inv_e = e == 0.f ? 0.f : 1.f / e;
    r.q_sum = e == 0.f ? 0.f : 1.f;
  }
  return r;
}

// The teacher's rest, against the student's mass off the list (`str` of `all`). One minus the sum of q is not zero where
// the slots hold everything: token_logprobs' log probabilities are off by 2^-20 + |t| 2^-22, which is (1 + H / 4) 2^-20 of
// the sum with H <= ln 128, and the exponentials and the sum add less than 1.2 2^-20. A rest below 2^-18 therefore counts
// as none where the student's probability of it is none either (below 2^-126): its term would be infinite, or 1e32 where
// the lowest value masks, from nothing but rounding.
__device__ __forceinline__ float rest_of(const Acc& str, const Acc& all, const ListStats& list, float c) {
  const float down = str.m == all.m ? 0.f : (str.m - all.m) * c;
  return list.q_rest <= 0x1p-18f && log2f(str.s) + down - log2f(all.s) < -126.f ? 0.f : list.q_rest;
}

// From the statistics of the streamed elements (all of them, or with TAIL those off the list).
template <bool TAIL>
__device__ __forceinline__ KdStats row_stats(const Acc& str, const ListStats& list, float c) {
  Acc all = str;
  if (TAIL) all.join<false>(list.z_max, list.z_sum, 0.f, c);
  KdStats r;
  r.t_max = list.t_max;
  r.inv_e = list.inv_e;
  r.m = all.m;
  r.inv_s = 1.f / all.s;
  // Where the student has no mass off the list, a rest is an infinite constant: it has no gradient.
  const float rest = TAIL ? rest_of(str, all, list, c) : 0.f;
  r.mass = TAIL && str.s != 0.f ? list.q_sum + rest : list.q_sum;
  r.coef = r.mass * r.inv_s;
  if (TAIL) {
    const float down = str.m == all.m ? 0.f : str.m - all.m;
    r.coef = str.s == 0.f ? 0.f : r.coef * ex2(down * c) - rest / str.s;
  }
  r.ms = str.m == -INFINITY ? 0.f : str.m;
  return r;
}

// The row's loss, by one warp.
template <bool TAIL>
__device__ __forceinline__ float row_loss(const Acc& str, const ListStats& list, const KdStats& r, float c, float inv_t,
                                          int K, const ListShared& sh) {
  const int lane = threadIdx.x & 31;
  Acc all = str;
  if (TAIL) all.join<false>(list.z_max, list.z_sum, 0.f, c);
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
  const float rest = TAIL ? rest_of(str, all, list, c) : 0.f;
  if (rest != 0.f) {
    const float down = str.m == all.m ? 0.f : str.m - all.m;
    loss += rest * (kLn2 * (log2f(rest) - log2f(str.s)) - down * inv_t + ln_s);
  }
  return loss;
}

// Gradient of the listed elements among units [u0, u1) and, if asked, the ragged ones: sums the q of slots that name
// the same token.
template <typename T>
__device__ __forceinline__ void write_listed(const Row<T>& row, T* out, int u0, int u1, bool ragged_too, int K, float c,
                                             float g, const KdStats& r, const ListShared& sh, int first, int step) {
  constexpr int E = Elem<T>::kUnit;
  for (int i = first; i < K; i += step) {
    const int id = sh.id[i];
    if (id < 0) continue;
    const int at = id - row.head;
    const bool in_body = at >= 0 && at < row.units * E;
    if (in_body ? !(at >= u0 * E && at < u1 * E) : !ragged_too) continue;
    float q = sh.q[i];
    if (sh.repeated) {
      q = 0.f;
      for (int j = 0; j < K; ++j)
        if (sh.id[j] == id) q += sh.q[j];
    }
    Elem<T>::store(out + id, g * (r.mass * (ex2((sh.z[i] - r.m) * c) * r.inv_s) - q));
  }
}

// Gradient of a row's units [u0, u1): the dense part in one pass, then the listed elements over it. The dense part stays
// in L2 till then: written past it, the scattered elements cost a read of their lines (16384 x 50257 bf16 with 64 slots:
// 573 against 535 us).
template <typename T, int NT, bool TAIL>
__device__ __forceinline__ void write_gradient(const Row<T>& row, T* out, int u0, int u1, int ragged, int K, float c,
                                               float g, const KdStats& r, ListShared& sh) {
  for (int i = threadIdx.x; i < K; i += NT) sh.q[i] = ex2((sh.t[i] - r.t_max) * (TAIL ? kLog2e : c)) * r.inv_e;
  const float dense = g * r.coef;
  const F2 minus_m = pair(-r.ms, -r.ms), cc = pair(c, c), dd = pair(dense, dense);
  map_row<T, NT, true>(row, out, u0, u1, ragged, [&](F2 z, int) {
    const float2 x = split(mul2(add2(z, minus_m), cc));
    return mul2(pair(ex2(x.x), ex2(x.y)), dd);
  });
  __syncthreads();
  write_listed<T>(row, out, u0, u1, ragged > 0, K, c, g, r, sh, threadIdx.x, NT);
}

// Loss of each row, times its weight: a block per row, or with SPLIT a cluster of blocks that share it. Off-list
// elements are told by marks in shared memory (TAIL). With GRAD, for short rows, a second pass over the row (from L2)
// writes the gradient.
template <typename T, int NT, bool TAIL, bool SPLIT, bool GRAD>
__global__ void __launch_bounds__(NT)
    distill_forward_kernel(const T* logits, long long ld, T* out, long long ld_out, int V,
                           const int64_t* __restrict__ ids, const float* __restrict__ teacher, int K, float c,
                           float inv_t, const float* __restrict__ weight, float* __restrict__ loss,
                           float* __restrict__ stats) {
  static_assert(!(SPLIT && GRAD), "a cluster leaves the gradient to the backward kernel");
  namespace cg = cooperative_groups;
  extern __shared__ uint32_t words[];
  __shared__ ListShared sh;
  __shared__ Acc join_sm[NT / 32], result;
  __shared__ KdStats row_result;
  const int tid = threadIdx.x;
  int part = 0, parts = 1;
  if constexpr (SPLIT) {
    part = (int)cg::this_cluster().block_rank();
    parts = (int)cg::this_cluster().num_blocks();
  }
  const long long row_i = SPLIT ? blockIdx.x / parts : blockIdx.x;
  const Row<T> row(logits + row_i * ld, V);
  int u0, u1;
  segment(row.units, part, parts, u0, u1);
  const int ragged = part == 0 ? row.ragged : 0;
  const float w = weight ? weight[row_i] : 1.f;
  const Marks<T, NT> marks(words, u0, u1);
  if (tid == 0) sh.repeated = 0;
  if (TAIL)
    for (int i = tid; i < Marks<T, NT>::size(u1 - u0); i += NT) words[i] = 0;
  const bool some = w != 0.f && __syncthreads_or(read_slots<T, NT>(row.z, V, ids + row_i * K, teacher + row_i * K, K, sh));
  if (!some) {
    if (part == 0 && tid == 0) loss[row_i] = 0.f;
    if (part == 0 && tid < kStats && stats) stats[row_i * kStats + tid] = 0.f;
    if constexpr (GRAD) {
      const Row<T> to(out + row_i * ld_out, V);
      zero_row<T, NT>(to, 0, to.units, to.ragged);
    }
    return;
  }
  Run<false> run;
  if (TAIL) {
    for (int i = tid; i < K; i += NT)
      if (sh.id[i] >= 0 && marks.mark(row, sh.id[i], part == 0)) sh.repeated = 1;
    __syncthreads();
  }
  if (tid < 32) {  // fewer than two units of ragged elements
    const bool in = tid < ragged && (!TAIL || !marks.ragged(tid));
    run.add_one(in ? Elem<T>::load(row.z + row.ragged_index(tid)) : -INFINITY, c);
  }
  const FromMemory src{row.unit_ptr()};
  if constexpr (TAIL) stream_units<T, NT, false>(src, u0, u1, c, run, marks, [](int, float) {});
  else stream_units<T, NT, false>(src, u0, u1, c, run, NoMarks{}, [](int, float) {});
  Acc all = block_join<NT>(run, c, join_sm);
  if constexpr (SPLIT) {
    if (tid == 0) {
      result = all;
      result.a = (float)sh.repeated;  // a block sees the marks of its part only
    }
    cg::this_cluster().sync();
    if (part == 0 && tid < 32) {
      all = *cg::this_cluster().map_shared_rank(&result, (tid & 7) < parts ? tid & 7 : 0);
      if (__any_sync(0xffffffffu, all.a != 0.f)) sh.repeated = 1;
      __syncwarp();
      all = join_lanes<8, false>((tid & 7) < parts ? all : Acc(), c);
    }
    cg::this_cluster().sync();  // the parts' statistics are read
  }
  if (part == 0 && tid < 32) {
    const ListStats list = list_stats<TAIL>(c, K, sh);
    const KdStats r = row_stats<TAIL>(all, list, c);
    if (GRAD && tid == 0) row_result = r;
    const float l = row_loss<TAIL>(all, list, r, c, inv_t, K, sh);
    if (tid == 0) {
      loss[row_i] = w * l;
      if (stats) store_stats(stats + row_i * kStats, r);
    }
  }
  if constexpr (GRAD) {
    if (!TAIL && tid == 0) sh.repeated = 1;  // not known
    __syncthreads();
    write_gradient<T, NT, TAIL>(row, out + row_i * ld_out, 0, row.units, row.ragged, K, c, w * inv_t, row_result, sh);
  }
}

// A row's units [0, ..) staged in shared memory.
struct FromStage {
  static constexpr bool kPatch = true;  // marked elements are put to -inf where they are
  uint4* stage;
  uint64_t* full;
  uint32_t phases;  // a chunk's parity each
  volatile int* abort_flag;
  int* status;
  // Waits for the batch's chunk to be there; a copy that does not arrive is recorded, and the host raises on it.
  __device__ __forceinline__ void begin(int batch) const {
    mbar_wait(&full[batch], (phases >> batch) & 1u, abort_flag, status, kStatusTimeoutRowStage);
  }
  __device__ __forceinline__ uint4 load(int u) const { return stage[u]; }
  template <typename T>
  __device__ __forceinline__ void patch(int u, int j) const {
    Elem<T>::store(reinterpret_cast<T*>(stage + u) + j, -INFINITY);
  }
};

// Loss and gradient of each row in one go: the logits are read from memory once and the gradient written once.
//
// A persistent block stages a row in shared memory by bulk copies, a chunk per barrier. Its streaming warps take the
// statistics in a first pass and write the gradient in a second; a chunk that all of them have left behind is filled
// with the block's next row at once, by a fetching warp. A serving warp joins the statistics and does all work on the
// lists: the next row's list is read, marked and summed during this row's second pass, and the listed elements are
// written after the dense gradient. Two blocks share an SM, so that one stores and fetches while the other is between
// its passes.
// 16384 x 50257 bf16 with 64 slots: 625 us with the rest, 596 without, 0.81 and 0.85 of the copy rate (up to 8 % more on
// some devices); issue slots and 2^x are busy 62 % of the time each. Reading the row twice through L2 instead took 849 us, more than two kernels
// (815 us): too many rows are in flight for L2 to hold them.
constexpr int kOwn = kMaxList / 32;  // slots per lane of the serving warp

struct GradShared {
  ListShared list[2];
  KdStats stats;
  float weight[2];
  int some[2], fetch[2];
  uint64_t full[kChunks], empty[kChunks], told[2], ready, joined, solved, done;
  int abort_flag;
};

template <typename T, int NT, bool TAIL>
__global__ void __launch_bounds__(NT + 64, 1024 / NT)
    distill_grad_kernel(const T* logits, long long ld, T* out, long long ld_out, int V, long long rows,
                        const int64_t* __restrict__ ids, const float* __restrict__ teacher, int K, float c, float inv_t,
                        const float* __restrict__ weight, float* __restrict__ loss, float* __restrict__ stats,
                        int stage_units, int* status) {
  extern __shared__ __align__(128) uint8_t dynamic[];
  constexpr int NW = NT / 32, kChunk = kBatch * NT;  // units of a batch of the streaming warps
  uint4* stage = reinterpret_cast<uint4*>(dynamic);
  uint32_t* words = reinterpret_cast<uint32_t*>(dynamic + 16 * (size_t)stage_units);
  __shared__ GradShared sh;
  __shared__ Acc sums[NW];
  const int tid = threadIdx.x, lane = tid & 31;
  const int chunks = (stage_units + kChunk - 1) / kChunk;
  if (tid == 0) {
    for (int i = 0; i < chunks; ++i) {
      mbar_init(&sh.full[i], 1);
      mbar_init(&sh.empty[i], NW);
    }
    mbar_init(&sh.told[0], 1);
    mbar_init(&sh.told[1], 1);
    mbar_init(&sh.ready, 1);
    mbar_init(&sh.joined, NW);
    mbar_init(&sh.solved, 1);
    mbar_init(&sh.done, NW + 1);
    sh.abort_flag = 0;
    fence_barrier_init();
  }
  for (int i = tid; i < Marks<T, NT>::size(stage_units); i += NT + 64) words[i] = 0;
  __syncthreads();
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    return mbar_wait(bar, parity & 1u, &sh.abort_flag, status, kStatusTimeoutRowStage);
  };
  // Rows so far, and for each chunk the parity of the rows that had units in it. Rows at other boundaries may end just
  // before the last chunk; they leave it alone, since no one would see it filled before it is given up. `told` completes
  // once per other row (one barrier for even rows and one for odd ones), the other barriers once per row. Each may
  // complete only after everyone who waits on it has seen it complete before: joined and solved(n + 1) follow done(n),
  // which needs every streaming warp to have seen solved(n); ready(n + 1) follows joined(n); told(n + 2) follows done(n),
  // which the fetching warp arrives on once it has seen told(n + 1). told(n + 1) follows nothing that the fetching warp
  // does in row n, so on one barrier it could complete twice before that warp looks.
  uint32_t count = 0, phases = 0;
  auto chunks_of = [&](const Row<T>& row) { return (row.units + kChunk - 1) / kChunk; };

  if (tid < NT) {
    for (long long r = blockIdx.x; r < rows; r += gridDim.x, ++count) {
      const Row<T> row(logits + r * ld, V);
      T* o = out + r * ld_out;
      const float rag = tid < row.ragged ? Elem<T>::load(row.z + row.ragged_index(tid)) : -INFINITY;
      wait(&sh.ready, count);
      const float g = sh.weight[count & 1] * inv_t;
      if (!sh.some[count & 1]) {
        if (lane == 0) mbar_arrive(&sh.joined);
        wait(&sh.solved, count);
        const Row<T> to(o, V);
        zero_row<T, NT>(to, 0, to.units, to.ragged);
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.done);
        continue;
      }
      Run<false> run;
      const FromStage src{stage, sh.full, phases, &sh.abort_flag, status};
      const Marks<T, NT> marks(words, 0, row.units);
      if (tid < 32) run.add_one(TAIL && tid < row.ragged && marks.ragged(tid) ? -INFINITY : rag, c);
      if constexpr (TAIL) stream_units<T, NT, false>(src, 0, row.units, c, run, marks, [](int, float) {});
      else stream_units<T, NT, false>(src, 0, row.units, c, run, NoMarks{}, [](int, float) {});
      const Acc mine = run.total(c);
      if (lane == 0) {
        sums[tid >> 5] = mine;
        mbar_arrive(&sh.joined);
      }
      wait(&sh.solved, count);
      const F2 minus_m = pair(-sh.stats.ms, -sh.stats.ms), cc = pair(c, c);
      const F2 dd = pair(g * sh.stats.coef, g * sh.stats.coef);
      auto gradient = [&](F2 v, int) {
        const float2 x = split(mul2(add2(v, minus_m), cc));
        return mul2(pair(ex2(x.x), ex2(x.y)), dd);
      };
      const bool same = same_boundaries(row.z, o);
      const int used = chunks_of(row);
      for (int i = 0; i < used; ++i) {
        map_batch<T, NT, true, false>(row, src, o, same, i * kChunk + tid, row.units, gradient, [&] {
          // The chunk's place is written by a bulk copy next, through another proxy: without the fence that copy could
          // overtake these loads (it did, for some hundred of 10^9 elements), and what was put to -inf.
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh.empty[i]);
        });
      }
      if (tid < row.ragged) Elem<T>::store(o + row.ragged_index(tid), split(gradient(pair(rag, 0.f), 0)).x);
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.done);
      phases ^= (1u << used) - 1u;
    }
    return;
  }

  if (tid < NT + 32) {
    // The fetching warp: told(n) says whether row n of this block has slots, or is behind
    // the last.
    bool open = true;
    for (long long r = blockIdx.x; open; r += gridDim.x, ++count) {
      if (!__all_sync(0xffffffffu, wait(&sh.told[count & 1], count >> 1))) break;
      const bool some = sh.fetch[count & 1];
      __syncwarp();
      if (lane == 0 && count > 0) mbar_arrive(&sh.done);  // of the row before
      if (r >= rows) return;
      if (!some) continue;
      const Row<T> row(logits + r * ld, V);
      const int used = chunks_of(row);
      for (int i = 0; i < used; ++i) {
        // Of the row before; a new barrier lets the first one pass.
        open = __all_sync(0xffffffffu, wait(&sh.empty[i], ~(phases >> i)));
        if (!open) break;
        if (lane == 0) {
          const uint32_t bytes = 16u * (uint32_t)min(kChunk, row.units - i * kChunk);
          mbar_arrive_expect_tx(&sh.full[i], bytes);
          bulk_load_1d(stage + i * kChunk, row.unit_ptr() + i * kChunk, bytes, &sh.full[i]);
        }
        phases ^= 1u << i;
        __syncwarp();
      }
    }
    // A wait ran out: no more is fetched, and what is on its way to this block's memory is waited for (with a limit).
    volatile int never = 0;
    for (int i = 0; i < chunks; ++i)
      if (!mbar_wait(&sh.full[i], ~(phases >> i) & 1u, &never, status, kStatusTimeoutDrain)) break;
    return;
  }

  // The serving warp. Slots lane, lane + 32, ... of the row that comes next:
  int64_t given[kOwn];
  float t[kOwn], z[kOwn], w = 0.f;
  auto ask = [&](long long r) {
    w = r < rows ? (weight ? weight[r] : 1.f) : 0.f;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      const bool in = r < rows && i * 32 + lane < K;
      given[i] = in ? ids[r * K + i * 32 + lane] : -1;
      t[i] = in ? teacher[r * K + i * 32 + lane] : 0.f;
    }
  };
  auto valid = [&](int i) { return given[i] >= 0 && given[i] < V; };
  auto ask_logits = [&](long long r) {
#pragma unroll
    for (int i = 0; i < kOwn; ++i) z[i] = valid(i) ? Elem<T>::load(logits + r * ld + given[i]) : 0.f;
  };
  auto any_slot = [&] {
    bool any = false;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) any |= valid(i);
    return __any_sync(0xffffffffu, any) && w != 0.f;
  };
  // Gives the row out to the streaming warps: its list, marks and what the list alone decides.
  auto prepare = [&](const Row<T>& row, uint32_t n, bool some) {
    ListShared& list = sh.list[n & 1];
    ListStats ls{};
    if (some) {
      if (lane == 0) list.repeated = 0;
      __syncwarp();
#pragma unroll
      for (int i = 0; i < kOwn; ++i) {
        if (i * 32 + lane < K) {
          const int id = valid(i) ? (int)given[i] : -1;
          list.id[i * 32 + lane] = id;
          list.t[i * 32 + lane] = valid(i) ? t[i] : -INFINITY;
          list.z[i * 32 + lane] = z[i];
          if (id >= 0 && Marks<T, NT>(words, 0, row.units).mark(row, id, true)) list.repeated = 1;
        }
      }
      __syncwarp();
      ls = list_stats<TAIL>(c, K, list);
    }
    if (lane == 0) {
      sh.some[n & 1] = some;
      sh.weight[n & 1] = w;
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh.ready);
    return ls;
  };
  auto tell = [&](uint32_t n, bool some) {
    if (lane == 0) {
      sh.fetch[n & 1] = some;
      mbar_arrive(&sh.told[n & 1]);
    }
    __syncwarp();
  };
  ask(blockIdx.x);
  bool some = any_slot();
  tell(0, some);
  ask_logits(blockIdx.x);
  ListStats list = prepare(Row<T>(logits + blockIdx.x * ld, V), 0, some);
  float w_now = w;
  ask(blockIdx.x + (long long)gridDim.x);
  for (long long r = blockIdx.x; r < rows; r += gridDim.x, ++count) {
    const long long next = r + gridDim.x;
    const Row<T> row(logits + r * ld, V), next_row(logits + (next < rows ? next : r) * ld, V);
    ListShared& now = sh.list[count & 1];
    const bool some_next = any_slot();
    tell(count + 1, some_next);
    ask_logits(next);
    KdStats k;
    Acc all;
    wait(&sh.joined, count);
    if (some) {
      all = join_lanes<NW, false>(sums[lane & (NW - 1)], c);
      k = row_stats<TAIL>(all, list, c);
      if (lane == 0) sh.stats = k;
    }
    if (lane == 0) mbar_arrive(&sh.solved);
    // The streaming warps are in the second pass, or write zeros.
    const ListStats list_now = list;
    if (some) {
      for (int i = lane; i < K; i += 32)
        if (now.id[i] >= 0) Marks<T, NT>(words, 0, row.units).unmark(row, now.id[i]);
      __syncwarp();
    }
    const float w_next = w;
    if (next < rows) list = prepare(next_row, count + 1, some_next);
    ask(next + gridDim.x);
    if (some) {
      const float l = row_loss<TAIL>(all, list_now, k, c, inv_t, K, now);
      if (lane == 0) {
        loss[r] = w_now * l;
        if (stats) store_stats(stats + r * kStats, k);
      }
      for (int i = lane; i < K; i += 32) now.q[i] = ex2((now.t[i] - k.t_max) * (TAIL ? kLog2e : c)) * k.inv_e;
    }
    wait(&sh.done, count);
    if (some) {
      __syncwarp();
      write_listed<T>(row, out + r * ld_out, 0, row.units, true, K, c, w_now * inv_t, k, now, lane, 32);
    } else {
      if (stats && lane < kStats) stats[r * kStats + lane] = 0.f;
      if (lane == 0) loss[r] = 0.f;
    }
    __syncwarp();
    some = some_next;
    w_now = w_next;
  }
}

// Gradient from the statistics the forward pass left; with `unless_one` nothing is done where the scale is one.
template <typename T, int NT, bool TAIL>
__global__ void __launch_bounds__(NT, 1280 / NT)
    distill_backward_kernel(const T* logits, long long ld, T* out, long long ld_out, int V, long long rows,
                            const int64_t* __restrict__ ids, const float* __restrict__ teacher, int K, float c,
                            float inv_t, const float* __restrict__ stats, RowGrad row_scale, const float* __restrict__ scale,
                            bool unless_one) {
  __shared__ ListShared sh;
  const float factor = scale ? *scale : 1.f;
  if (unless_one && factor == 1.f) return;
  for (long long i = blockIdx.x; i < rows; i += gridDim.x) {
    const long long row_i = rows - 1 - i;  // last rows first: the forward pass left them in L2
    const float* s = stats + row_i * kStats;
    const float w = row_scale.at(row_i, 1.f);
    T* o = out + row_i * ld_out;
    int u0, u1;
    if (s[7] == 0.f || w == 0.f) {
      const Row<T> row(o, V);
      segment(row.units, blockIdx.y, gridDim.y, u0, u1);
      zero_row<T, NT>(row, u0, u1, blockIdx.y == 0 ? row.ragged : 0);
      continue;
    }
    const Row<T> row(logits + row_i * ld, V);
    segment(row.units, blockIdx.y, gridDim.y, u0, u1);
    const KdStats r{s[0], s[1], s[2], s[3], s[4], s[5], s[6]};
    if (threadIdx.x == 0) sh.repeated = 1;  // not known here
    read_slots<T, NT>(row.z, V, ids + row_i * K, teacher + row_i * K, K, sh);
    if (o == row.z) __syncthreads();  // the listed logits are read before the gradient takes their place
    write_gradient<T, NT, TAIL>(row, o, u0, u1, blockIdx.y == 0 ? row.ragged : 0, K, c, w * factor * inv_t, r, sh);
    __syncthreads();  // the list is read before the next row's replaces it
  }
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
                               const OptTensor& weight, const at::Tensor& loss, const OptTensor& stats,
                               const OptTensor& out, int64_t vocab, double temperature, bool tail) {
  const int64_t rows = check_logits(logits, vocab, temperature, "logits");
  const int k = check_teacher(ids, teacher, rows, logits);
  if (weight) check_rows(*weight, "weight", rows, 1, at::kFloat, logits);
  check_rows(loss, "loss", rows, 1, at::kFloat, logits);
  if (stats) check_rows(*stats, "stats", rows, kStats, at::kFloat, logits);
  if (out) check_out(*out, logits, vocab);
  if (rows == 0) return;
  const int device = logits.get_device();
  // Loss and gradient in one kernel: rows of up to 32 KB pass twice through L2, and others are staged where they fit into
  // half an SM's shared memory and fill the device. The rest takes two kernels.
  const int64_t row_bytes = vocab * logits.element_size(), units = row_bytes / 16;
  const int stage_units = (int)((units + 7) / 8 * 8);
  const int64_t staged = 16 * (int64_t)stage_units + 4 * Marks<__half, kGradThreads>::size(stage_units);
  const bool twice = out && row_bytes <= 32 * 1024;
  const bool together = out && !twice && staged <= kStageBytes && rows >= num_sms(device);
  if (out && !twice && !together) {
    KB_CHECK(stats.has_value(), "the gradient needs stats");
    topk_distillation_forward(logits, ids, teacher, weight, loss, stats, c10::nullopt, vocab, temperature, tail);
    topk_distillation_backward(logits, ids, teacher, *stats, weight, c10::nullopt, *out, vocab, temperature, tail, false);
    return;
  }
  const c10::cuda::CUDAGuard guard(logits.device());
  cudaStream_t s = c10::cuda::getCurrentCUDAStream().stream();
  const float c = (float)(1.4426950408889634 / temperature), inv_t = (float)(1.0 / temperature);
  const float* w = weight ? weight->data_ptr<float>() : nullptr;
  float* kept = stats ? stats->data_ptr<float>() : nullptr;
  for_logits_type(logits.scalar_type(), [&](auto tag) {
    using T = typename decltype(tag)::type;
    for_bool(tail, [&](auto tail_tag) {
      constexpr bool TAIL = decltype(tail_tag)::value;
      if (together) {
        auto kern = distill_grad_kernel<T, kGradThreads, TAIL>;
        const int per_sm = allow_smem(kern, (size_t)staged, kGradThreads + 64, device);
        const int64_t blocks = std::min<int64_t>(rows, (int64_t)std::max(1, per_sm) * compute_sms(device));
        launch_rows(kern, blocks, kGradThreads + 64, 1, (size_t)staged, s, (const T*)logits.data_ptr(), logits.stride(0),
                    (T*)out->data_ptr(), out->stride(0), (int)vocab, rows, ids.data_ptr<int64_t>(),
                    teacher.data_ptr<float>(), k, c, inv_t, w, loss.data_ptr<float>(), kept, stage_units,
                    device_status_ptr(device));
        return;
      }
      if (twice) {
        constexpr int NT = 128;
        launch_rows(distill_forward_kernel<T, NT, TAIL, false, true>, rows, NT, 1,
                    TAIL ? 4 * (size_t)Marks<T, NT>::size((int)units) : 0, s, (const T*)logits.data_ptr(),
                    logits.stride(0), (T*)out->data_ptr(), out->stride(0), (int)vocab, ids.data_ptr<int64_t>(),
                    teacher.data_ptr<float>(), k, c, inv_t, w, loss.data_ptr<float>(), kept);
        return;
      }
      const RowLaunch how = row_launch(rows, vocab * (int64_t)sizeof(T), true, device);
      for_row_launch(how, [&](auto nt_tag, auto split_tag) {
        constexpr int NT = decltype(nt_tag)::value;
        auto kern = distill_forward_kernel<T, NT, TAIL, decltype(split_tag)::value, false>;
        const int smem = TAIL ? 4 * Marks<T, NT>::size((int)((units + how.parts - 1) / how.parts)) : 0;
        if (smem > 32 * 1024) allow_smem(kern, (size_t)smem, 0, device);
        launch_rows(kern, rows, NT, how.parts, (size_t)smem, s, (const T*)logits.data_ptr(), logits.stride(0), nullptr,
                    0, (int)vocab, ids.data_ptr<int64_t>(), teacher.data_ptr<float>(), k, c, inv_t, w,
                    loss.data_ptr<float>(), kept);
      });
    });
  });
  KB_LAUNCHED();
}

void topk_distillation_backward(const at::Tensor& logits, const at::Tensor& ids, const at::Tensor& teacher,
                                const at::Tensor& stats, const OptTensor& row_scale, const OptTensor& scale,
                                const at::Tensor& out, int64_t vocab, double temperature, bool tail, bool unless_one) {
  const int64_t rows = check_logits(logits, vocab, temperature, "logits");
  check_out(out, logits, vocab);
  const int k = check_teacher(ids, teacher, rows, logits);
  check_rows(stats, "stats", rows, kStats, at::kFloat, logits);
  const RowGrad row_grad = check_row_grad(row_scale, "row_scale", rows, logits);
  if (scale) check_rows(*scale, "scale", 1, 1, at::kFloat, logits);
  if (rows == 0) return;
  const c10::cuda::CUDAGuard guard(logits.device());
  cudaStream_t s = c10::cuda::getCurrentCUDAStream().stream();
  const float c = (float)(1.4426950408889634 / temperature);
  for_logits_type(logits.scalar_type(), [&](auto tag) {
    using T = typename decltype(tag)::type;
    const int nseg = row_segments(rows, vocab, sizeof(T), 256, logits.get_device());
    // Blocks that most often return at once are few, and take several rows where they do not.
    const int64_t blocks = unless_one ? std::min<int64_t>(rows, 8 * (int64_t)num_sms(logits.get_device())) : rows;
    for_bool(tail, [&](auto tail_tag) {
      const bool small = vocab * (int64_t)sizeof(T) <= kSmallRow;
      const auto kern = small ? distill_backward_kernel<T, 64, decltype(tail_tag)::value>
                              : distill_backward_kernel<T, 256, decltype(tail_tag)::value>;
      kern<<<dim3((unsigned)blocks, nseg), small ? 64 : 256, 0, s>>>(
          (const T*)logits.data_ptr(), logits.stride(0), (T*)out.data_ptr(), out.stride(0), (int)vocab, rows,
          ids.data_ptr<int64_t>(), teacher.data_ptr<float>(), k, c, (float)(1.0 / temperature),
          stats.data_ptr<float>(), row_grad,
          scale ? scale->data_ptr<float>() : nullptr, unless_one);
    });
  });
  KB_LAUNCHED();
}

void register_topk_distillation_ops(pybind11::module& m) {
  m.def("topk_distillation_forward", &topk_distillation_forward, "KL divergence from a teacher's top logits");
  m.def("topk_distillation_backward", &topk_distillation_backward, "gradient of topk_distillation_forward");
  m.attr("TOPK_DISTILLATION_STATS") = kStats;
}

}  // namespace kb
