// Log probabilities of given tokens, with the entropy of each row's
// distribution and its most likely alternatives, and their gradient.
#include <torch/csrc/utils/pybind.h>

#include "token_losses.cuh"

namespace kb {
namespace {

constexpr int kCand = 512;   // candidates held while the alternatives are selected
constexpr int kStats = kTokenLogprobsStats;  // m, log2 S

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

constexpr int kHits = 256;  // units looked at element by element

template <int NT>
struct SelectShared {
  static constexpr int kGroups = NT == 256 ? 16 : 8;  // maxima kept per thread: batch b counts to group b % kGroups
  union alignas(16) {
    float group_max[kGroups][NT];
    unsigned long long cand[kCand];
    unsigned long long merged[8 * kMaxTopK];  // the sorted lists of a cluster's blocks
  };
  union {
    uint16_t list[kGroups * NT];
    int sums[NT / 32];  // counts per warp
  };
  union {
    uint4 hit[kHits];
    uint32_t list_key[4 * kHits];  // maxima of the first listed groups
  };
  int hit_unit[kHits];
  uint32_t warp_key[NT / 32], warp_top[NT / 32];
  int count, listed, hits;
};

// Calls emit(i, key) for the k largest keys of a block's elements, i their
// places in descending order (fewer where the block has fewer elements).
//
// Selection without a second pass over the row: the statistics' pass keeps
// the maximum of each thread, and of each group of a thread's batches.
// 1. With r = k / warps, rounded up, let t be the least of the (full) warps'
//    r-th largest thread maxima: at least k elements are >= t.
// 2. One warp bisects t among those groups' maxima until not many more than k
//    are left. All k largest elements are >= t still, and lie in these groups.
// 3. Those groups are read again (from L2), first for the units with an
//    element >= t, then for the elements, which are ranked by counting.
// Ties and rows sorted in memory can make the candidates overflow; then the
// k-th value is bisected over the row itself and ties are taken in index order.
template <typename T, int NT, typename Emit>
__device__ void select_top(const Row<T>& row, int u0, int u1, int ragged, float mine, int k, int few,
                           SelectShared<NT>& sh, const Emit& emit) {
  constexpr int E = Elem<T>::kUnit, NW = NT / 32, kGroups = SelectShared<NT>::kGroups;
  static_assert(NW <= 32 && NT * kGroups <= 65536, "list entries are 16 bits wide");
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n_units = u1 - u0;
  const int want = min(k, n_units * E + ragged);
  const bool has = tid < n_units || tid < ragged;
  const uint32_t key = has ? order_of(mine) : 0u;
  const int warps = min(NW, n_units / 32);  // all of whose lanes have elements
  const int r = warps > 0 ? (want + warps - 1) / warps : 33;
  {
    // The warp's r-th largest: take the maximum out until r are gone.
    uint32_t rest = key, top = 0;
    int gone = 0;
    while (gone < min(r, 32)) {
      top = __reduce_max_sync(0xffffffffu, rest);
      if (lane == 0 && gone == 0) sh.warp_top[warp] = top;
      gone = top == 0 ? 32 : gone + __popc(__ballot_sync(0xffffffffu, rest == top));
      rest = rest == top ? 0u : rest;
    }
    if (lane == 0) sh.warp_key[warp] = top;
  }
  if (tid == 0) {
    sh.count = 0;
    sh.listed = 0;
    sh.hits = 0;
  }
  __syncthreads();
  // Where the warps have too few lanes all elements stay: no key is 0.
  uint32_t t = __reduce_min_sync(0xffffffffu, lane < warps ? sh.warp_key[lane] : 0xFFFFFFFFu);
  t = r > 32 ? 1u : t;
  const uint32_t top = __reduce_max_sync(0xffffffffu, sh.warp_top[lane & (NW - 1)]);
  const int batches = (n_units + kBatch * NT - 1) / (kBatch * NT);
  // Candidates are told by their values first: !(v < bound) holds for all of order >= t, and for NaN.
  float bound = value_of(t);
  if (key >= t) {
    for (int g = 0; g < min(batches, kGroups); ++g) {
      const float m = sh.group_max[g][tid];
      if (tid + g * kBatch * NT >= n_units || m < bound) continue;
      const int at = atomicAdd(&sh.listed, 1);
      sh.list[at] = (uint16_t)(g * NT + tid);
      if (at < 4 * kHits) sh.list_key[at] = order_of(m);
    }
  }
  __syncthreads();
  const int listed = sh.listed;
  // Where blocks are few and latency counts, some more than enough are looked at all the same.
  if (listed > max(few, want + want / 8 + 2) && listed <= 4 * kHits) {
    if (warp == 0) {
      uint32_t lo = t, hi = top;  // count(>= lo) >= want, count(> hi) < want
      while (lo < hi) {
        const uint32_t mid = lo + (hi - lo) / 2 + 1;
        int n = 0;
        for (int i = lane; i < listed; i += 32) n += sh.list_key[i] >= mid;
        n = __reduce_add_sync(0xffffffffu, n);
        if (n >= want) {
          lo = mid;
          if (n <= want + want / 8 + 2) break;
        } else {
          hi = mid - 1;
        }
      }
      if (lane == 0) sh.warp_key[0] = lo;
    }
    __syncthreads();
    t = sh.warp_key[0];
    bound = value_of(t);
  }
  auto push = [&](float v, int idx) {
    if (v < bound) return;
    const uint32_t o = order_of(v);
    if (o < t) return;
    const int at = atomicAdd(&sh.count, 1);
    if (at < kCand) sh.cand[at] = key_of(o, idx);
  };
  const uint4* p = row.unit_ptr();
  for (int first = 0; first < batches; first += kGroups) {
    for (int i = tid; i < listed * kBatch; i += NT) {
      const int entry = sh.list[i / kBatch];
      const int u = u0 + entry % NT + ((entry / NT + first) * kBatch + i % kBatch) * NT;
      if (u < u1 && !(sh.group_max[entry / NT][entry % NT] < bound)) {
        const uint4 q = load_unit(p + u);
        const float mx = Elem<T>::widen_max(Elem<T>::max2(Elem<T>::max2(q.x, q.y), Elem<T>::max2(q.z, q.w)));
        if (!(mx < bound)) {
          const int at = atomicAdd(&sh.hits, 1);
          if (at < kHits) {
            sh.hit[at] = q;
            sh.hit_unit[at] = u;
          }
        }
      }
    }
  }
  __syncthreads();
  const int hits = min(sh.hits, kHits);
  if (tid < ragged) push(Elem<T>::load(row.z + row.ragged_index(tid)), row.ragged_index(tid));
  for (int i = tid; i < hits * E; i += NT)
    push(Elem<T>::load(reinterpret_cast<const T*>(sh.hit) + i), row.head + sh.hit_unit[i / E] * E + i % E);
  __syncthreads();
  int n = sh.hits > kHits ? kCand + 1 : sh.count;
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
      if (lane == 0) sh.sums[warp] = __popc(vote);
      __syncthreads();
      int before = taken, sum = 0;
      for (int w = 0; w < NT / 32; ++w) {
        if (w < warp) before += sh.sums[w];
        sum += sh.sums[w];
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
    int j = 0;
#pragma unroll 4
    for (; j + 1 < n; j += 2) {
      const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(&sh.cand[j]);
      rank += (two.x > ki) + (two.y > ki);
    }
    if (j < n) rank += sh.cand[j] > ki;
    if (rank < want) emit(rank, ki);
  }
}

// --------------------------------------------------- log probabilities

// Statistics of a set of elements, told apart from those of the one thread that has more than half of the sum, if one
// has (owner >= 0): `own` is its sum to all.m, `others` the rest's statistics. Only there can the set have an element
// more likely than all others together.
struct Apart {
  Acc all, others;
  float own = 0.f;
  int owner = -1;
};
struct WarpStats {
  Acc others;
  float s = 0.f, a = 0.f;  // of the lane with more than half of the warp's sum
  int lane = 0;
};

__device__ __forceinline__ WarpStats warp_apart(const Run<true>& run, float c) {
  const float2 ss = split(run.s), aa = split(run.a);
  const float off = run.offset(c), f = ex2(-off);
  const float s = (ss.x + ss.y) * f, a = (aa.x + aa.y) * f - off * s;
  WarpStats w;
  w.others.m = run.m;
  w.others.s = warp_sum(s);
  const uint32_t most = __ballot_sync(0xffffffffu, 2.f * s > w.others.s);
  if (most) {
    w.lane = __ffs(most) - 1;
    w.s = __shfl_sync(0xffffffffu, s, w.lane);
    w.a = __shfl_sync(0xffffffffu, a, w.lane);
  }
  const bool apart = most && (int)(threadIdx.x & 31) == w.lane;
  if (most) w.others.s = warp_sum(apart ? 0.f : s);
  w.others.a = warp_sum(apart ? 0.f : a);
  return w;
}

// Joins the parts that the first N lanes of a warp hold: `owner` of its part, and the part's lane.
template <int N>
__device__ __forceinline__ Apart join_apart(const Acc& all, const Acc& others, float own, int owner, float c, int& part) {
  Apart r;
  r.all = join_lanes<N, true>(all, c);
  const bool mine = (int)(threadIdx.x & 31) < N;
  const float mass = mine && owner >= 0 ? own * (all.m == r.all.m ? 1.f : ex2((all.m - r.all.m) * c)) : 0.f;
  const uint32_t most = __ballot_sync(0xffffffffu, 2.f * mass > r.all.s);
  if (most) {
    part = __ffs(most) - 1;
    r.own = __shfl_sync(0xffffffffu, mass, part);
    r.owner = __shfl_sync(0xffffffffu, owner, part);
    const bool apart = (int)(threadIdx.x & 31) == part;
    Acc rest;
    rest.m = all.m;
    rest.s = apart ? others.s : all.s;
    rest.a = apart ? others.a : all.a;
    if (apart) rest.m = others.m;
    r.others = join_lanes<N, true>(rest, c);
  }
  return r;
}

// The same for a block's warps; the first warp returns with it.
template <int NT>
__device__ __forceinline__ Apart block_apart(const Run<true>& run, float c, WarpStats* sm) {
  const WarpStats mine = warp_apart(run, c);
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = mine;
  __syncthreads();
  Apart r;
  if (threadIdx.x < 32) {
    const WarpStats w = sm[threadIdx.x & (NT / 32 - 1)];
    Acc all = w.others;
    all.s += w.s;
    all.a += w.a;
    int warp = 0;
    r = join_apart<NT / 32>(all, w.others, w.s, w.lane, c, warp);
    if (r.owner >= 0) r.owner += 32 * warp;
  }
  return r;
}

// A block per row, or with SPLIT a cluster of blocks that share it: statistics
// in one pass, then the alternatives. The blocks of a cluster select their own
// alternatives, and the first block merges the sorted lists.
template <typename T, int NT, bool TOPK, bool SPLIT>
__global__ void __launch_bounds__(NT, 1280 / NT)
    logprob_forward_kernel(const T* __restrict__ logits, long long ld, int V, const int64_t* __restrict__ tokens,
                           int64_t ignore_index, float c, float inv_t, int k, float* __restrict__ logprobs,
                           float* __restrict__ entropy, float* __restrict__ stats, float* __restrict__ top_logprobs,
                           int64_t* __restrict__ top_ids) {
  namespace cg = cooperative_groups;
  const int tid = threadIdx.x;
  int part = 0, parts = 1;
  if constexpr (SPLIT) {
    part = (int)cg::this_cluster().block_rank();
    parts = (int)cg::this_cluster().num_blocks();
  }
  const long long row_i = SPLIT ? blockIdx.x / parts : blockIdx.x;
  const int64_t token = tokens ? tokens[row_i] : 0;
  if (tokens && token == ignore_index) {
    if (part == 0) {
      if (tid == 0) {
        logprobs[row_i] = 0.f;
        entropy[row_i] = 0.f;
        if (stats) stats[kStats * row_i] = stats[kStats * row_i + 1] = 0.f;
      }
      for (int i = tid; TOPK && i < k; i += NT) {
        top_logprobs[row_i * k + i] = 0.f;
        top_ids[row_i * k + i] = -1;
      }
    }
    return;
  }
  const Row<T> row(logits + row_i * ld, V);
  int u0, u1;
  segment(row.units, part, parts, u0, u1);
  const int ragged = part == 0 ? row.ragged : 0;
  Run<true> run;
  float mine = -INFINITY;
  if (tid < 32) {  // fewer than two units of ragged elements
    mine = tid < ragged ? Elem<T>::load(row.z + row.ragged_index(tid)) : -INFINITY;
    run.add_one(mine, c);
  }
  __shared__ WarpStats join_sm[NT / 32];
  __shared__ Acc result;
  __shared__ Apart mine_apart;
  __shared__ float star_logp;
  __shared__ int star;
  __shared__ std::conditional_t<TOPK, SelectShared<NT>, int> sh;
  stream_units<T, NT, TOPK>(FromMemory{row.unit_ptr()}, u0, u1, c, run, NoMarks{}, [&](int batch, float mx) {
    if constexpr (TOPK) {
      mine = max_nan(mine, mx);
      float& kept = sh.group_max[batch % sh.kGroups][tid];
      kept = batch < sh.kGroups ? mx : max_nan(kept, mx);
    }
  });
  const int per = (row.units + parts - 1) / parts;
  Apart got = block_apart<NT>(run, c, join_sm);
  int owner_part = 0;
  if constexpr (SPLIT) {
    __shared__ unsigned long long sorted[TOPK ? kMaxList : 1];
    if (tid == 0) mine_apart = got;
    if constexpr (TOPK) {
      for (int i = tid; i < k; i += NT) sorted[i] = 0;  // below every key
      select_top<T, NT>(row, u0, u1, ragged, mine, k, 64, sh,
                        [&](int place, unsigned long long key) { sorted[place] = key; });
    }
    cg::this_cluster().sync();
    if (part == 0) {
      if (tid < 32) {
        Apart theirs;
        if ((tid & 31) < parts) theirs = *cg::this_cluster().map_shared_rank(&mine_apart, tid & 7);
        got = join_apart<8>(theirs.all, theirs.others, theirs.own, theirs.owner, c, owner_part);
      }
      if constexpr (TOPK) {
        for (int i = tid; i < parts * k; i += NT) sh.merged[i] = *cg::this_cluster().map_shared_rank(&sorted[i % k], i / k);
      }
    }
    cg::this_cluster().sync();  // the other blocks' shared memory is not needed any more
    if (part != 0) return;
  }
  // Log probabilities are taken in units of z / T, not of c z: (lowest - m) c would overflow.
  if (tid < 32) {
    const Acc all = got.all;
    const float log2s = log2f(all.s);
    float logp = NAN, h = kLn2 * (log2s - all.a / all.s);
    if (tokens && token >= 0 && token < V)
      logp = (Elem<T>::load(row.z + token) - all.m) * inv_t - kLn2 * log2s;
    int best = -1;
    float best_logp = 0.f;
    if (got.owner >= 0) {
      // An element more likely than all others together: its ln p and the entropy are small differences of large numbers,
      // unless they are taken from the rest of the sum, -ln p = ln(1 + rest / e) and
      // H = -ln p - sum over the rest of p_j ln 2 (x_j - x). What its thread has added to the sum is summed anew.
      const int first = owner_part * per + got.owner, last = min(row.units, (owner_part + 1) * per);
      const int mine_u = first + tid * NT;  // the lane's only unit where a thread has at most 32
      uint4 q = make_uint4(0, 0, 0, 0);
      if (mine_u < last) q = load_unit(row.unit_ptr() + mine_u);
      const auto each = [&](const auto& take) {
        for (int u = mine_u; u < last; u += 32 * NT) {
          float v[Elem<T>::kUnit];
          Elem<T>::unpack(u == mine_u ? q : load_unit(row.unit_ptr() + u), v);
#pragma unroll
          for (int j = 0; j < Elem<T>::kUnit; ++j) take(v[j], row.head + u * Elem<T>::kUnit + j);
        }
        if (tid == 0 && owner_part == 0 && got.owner < row.ragged) {
          const int i = row.ragged_index(got.owner);
          take(Elem<T>::load(row.z + i), i);
        }
      };
      float z = -INFINITY;
      int at = 0x7FFFFFFF;
      each([&](float v, int i) {
        at = v > z || (v == z && i < at) ? i : at;
        z = fmaxf(z, v);
      });
      const float most = warp_max_nan(z), x = (most - all.m) * c, e = ex2(x);
      at = __reduce_min_sync(0xffffffffu, z == most ? at : 0x7FFFFFFF);
      if (2.f * e > all.s) {
        Acc rest;
        rest.m = all.m;
        each([&](float v, int i) {
          if (i == at) return;
          const float y = (v - all.m) * c, f = ex2(y);
          rest.s += f;
          rest.a = fmaf(f, fmaxf(y, -256.f), rest.a);
        });
        rest.s = warp_sum(rest.s);
        rest.a = warp_sum(rest.a);
        rest.join<true>(got.others.m, got.others.s, got.others.a, c);
        const float l = log1pf(rest.s / e);
        best = at;
        best_logp = -l;
        h = l - kLn2 * (rest.a - x * rest.s) / (rest.s + e);
        if (tokens && token == at) logp = -l;
      }
    }
    if (tid == 0) {
      if (tokens) logprobs[row_i] = logp;
      entropy[row_i] = h;
      if (stats) {
        stats[kStats * row_i] = all.m;
        stats[kStats * row_i + 1] = log2s;
      }
      if (TOPK) {
        result.m = all.m;
        result.s = kLn2 * log2s;
        star = best;
        star_logp = best_logp;
      }
    }
  }
  if constexpr (TOPK) {
    auto emit = [&](int place, unsigned long long key) {
      const int id = (int)~(uint32_t)key;
      top_ids[row_i * k + place] = id;
      top_logprobs[row_i * k + place] =
          id == star ? star_logp : (value_of((uint32_t)(key >> 32)) - result.m) * inv_t - result.s;
    };
    if constexpr (SPLIT) {
      __syncthreads();
      // A key's place is the number of larger keys: counted, or from its place in its own list and searches in the others.
      for (int i = tid; i < parts * k; i += NT) {
        const unsigned long long key = sh.merged[i];
        int place = 0;
        if (parts * k <= 128) {
          for (int j = 0; j < parts * k; ++j) place += sh.merged[j] > key;
        } else {
          place = i % k;
          for (int other = 0; other < parts; ++other) {
            if (other == i / k) continue;
            int lo = 0, hi = k;  // keys before lo are larger, from hi on smaller
            while (lo < hi) {
              const int mid = (lo + hi) / 2;
              if (sh.merged[other * k + mid] > key) lo = mid + 1;
              else hi = mid;
            }
            place += lo;
          }
        }
        if (key != 0 && place < k) emit(place, key);
      }
    } else {
      select_top<T, NT>(row, u0, u1, ragged, mine, k, NT == 512 ? 64 : 0, sh, emit);
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
                            RowGrad dlogprobs, RowGrad dentropy) {
  const long long row_i = gridDim.x - 1 - blockIdx.x;  // last rows first: the forward pass left them in L2
  const int64_t token = tokens ? tokens[row_i] : -1;
  float g = dlogprobs.at(row_i, 0.f);
  const float gh = dentropy.at(row_i, 0.f);
  int u0, u1;
  if ((tokens && token == ignore_index) || (g == 0.f && gh == 0.f)) {
    const Row<T> row(out + row_i * ld_out, V);
    segment(row.units, blockIdx.y, gridDim.y, u0, u1);
    zero_row<T, NT>(row, u0, u1, blockIdx.y == 0 ? row.ragged : 0);
    return;
  }
  if (token < 0 || token >= V) g = g == 0.f ? 0.f : NAN;  // its log probability is NaN too
  const Row<T> row(logits + row_i * ld, V);
  segment(row.units, blockIdx.y, gridDim.y, u0, u1);
  const float m = stats[kStats * row_i], log2s = stats[kStats * row_i + 1];
  const float a = -(g + gh * entropy[row_i]) * inv_t, b = -gh * kLn2 * inv_t, hot = g * inv_t;
  const int at = (int)token;
  T* o = out + row_i * ld_out;
  const int ragged = blockIdx.y == 0 ? row.ragged : 0;
  const F2 minus_m = pair(-m, -m), cc = pair(c, c), ml = pair(-log2s, -log2s), aa = pair(a, a), bb = pair(b, b);
  auto given = [&](F2 d, int j) {
    if ((unsigned)(at - j) < 2u) {
      const float2 s = split(d);
      d = at == j ? pair(s.x + hot, s.y) : pair(s.x, s.y + hot);
    }
    return d;
  };
  if (b == 0.f) {
    map_row<T, NT, false>(row, o, u0, u1, ragged, [&](F2 z, int j) {
      const float2 y = split(fma2(add2(z, minus_m), cc, ml));
      return given(mul2(pair(ex2(y.x), ex2(y.y)), aa), j);
    });
  } else {
    map_row<T, NT, false>(row, o, u0, u1, ragged, [&](F2 z, int j) {
      float2 y = split(fma2(add2(z, minus_m), cc, ml));
      const F2 p = pair(ex2(y.x), ex2(y.y));
      return given(mul2(p, fma2(bb, pair(fmaxf(y.x, -256.f), fmaxf(y.y, -256.f)), aa)), j);  // 0 (-inf) is 0 here
    });
  }
}

}  // namespace

void token_logprobs_forward(const at::Tensor& logits, const OptTensor& tokens, const OptTensor& logprobs,
                            const at::Tensor& entropy, const OptTensor& stats, const OptTensor& top_logprobs,
                            const OptTensor& top_ids, int64_t vocab, double temperature, int64_t ignore_index) {
  const int64_t rows = check_logits(logits, vocab, temperature, "logits");
  KB_CHECK(tokens.has_value() == logprobs.has_value(), "tokens and logprobs go together");
  KB_CHECK(top_logprobs.has_value() == top_ids.has_value(), "top_logprobs and top_ids go together");
  if (tokens) check_rows(*tokens, "tokens", rows, 1, at::kLong, logits);
  if (logprobs) check_rows(*logprobs, "logprobs", rows, 1, at::kFloat, logits);
  check_rows(entropy, "entropy", rows, 1, at::kFloat, logits);
  if (stats) check_rows(*stats, "stats", rows, kStats, at::kFloat, logits);
  int k = 0;
  if (top_ids) {
    KB_CHECK(top_ids->dim() >= 1, "top_ids must be [rows, k]");
    KB_CHECK(top_ids->size(-1) >= 1 && top_ids->size(-1) <= std::min<int64_t>(kMaxList, vocab),
             "1 to 128 alternatives, and no more than the vocabulary holds");
    k = (int)top_ids->size(-1);
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
    const RowLaunch how = row_launch(rows, vocab * (int64_t)sizeof(T), false, logits.get_device());
    for_bool(k > 0, [&](auto top_tag) {
      for_row_launch(how, [&](auto nt_tag, auto split_tag) {
        constexpr int NT = decltype(nt_tag)::value;
        launch_rows(logprob_forward_kernel<T, NT, decltype(top_tag)::value, decltype(split_tag)::value>, rows, NT,
                    how.parts, 0, s, (const T*)logits.data_ptr(), logits.stride(0), (int)vocab, tok, ignore_index, c,
                    (float)(1.0 / temperature), k, lp, entropy.data_ptr<float>(), stats ? stats->data_ptr<float>() : nullptr,
                    tl, ti);
      });
    });
  });
  KB_LAUNCHED();
}

void token_logprobs_backward(const at::Tensor& logits, const OptTensor& tokens, const at::Tensor& stats,
                             const at::Tensor& entropy, const OptTensor& dlogprobs, const OptTensor& dentropy,
                             const at::Tensor& out, int64_t vocab, double temperature, int64_t ignore_index) {
  const int64_t rows = check_logits(logits, vocab, temperature, "logits");
  check_out(out, logits, vocab);
  if (tokens) check_rows(*tokens, "tokens", rows, 1, at::kLong, logits);
  KB_CHECK(tokens.has_value() || !dlogprobs.has_value(), "dlogprobs without tokens");
  check_rows(stats, "stats", rows, kStats, at::kFloat, logits);
  check_rows(entropy, "entropy", rows, 1, at::kFloat, logits);
  const RowGrad dlp = check_row_grad(dlogprobs, "dlogprobs", rows, logits);
  const RowGrad dh = check_row_grad(dentropy, "dentropy", rows, logits);
  if (rows == 0) return;
  const c10::cuda::CUDAGuard guard(logits.device());
  cudaStream_t s = c10::cuda::getCurrentCUDAStream().stream();
  const float c = (float)(1.4426950408889634 / temperature);
  for_logits_type(logits.scalar_type(), [&](auto tag) {
    using T = typename decltype(tag)::type;
    const int nseg = row_segments(rows, vocab, sizeof(T), 256, logits.get_device());
    const bool small = vocab * (int64_t)sizeof(T) <= kSmallRow;
    const auto kern = small ? logprob_backward_kernel<T, 64> : logprob_backward_kernel<T, 256>;
    kern<<<dim3((unsigned)rows, nseg), small ? 64 : 256, 0, s>>>(
        (const T*)logits.data_ptr(), logits.stride(0), (T*)out.data_ptr(), out.stride(0), (int)vocab,
        tokens ? tokens->data_ptr<int64_t>() : nullptr, ignore_index, c, (float)(1.0 / temperature),
        stats.data_ptr<float>(), entropy.data_ptr<float>(), dlp, dh);
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
