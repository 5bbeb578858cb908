// Device and host pieces shared by the per-token losses over a vocabulary
// (token_logprobs.cu, topk_distillation.cu).
//
// Notation: z is a row of V logits, c = log2(e) / T, m = max z,
// S = sum_j 2^((z_j - m) c), so p_j = 2^((z_j - m) c) / S is softmax(z / T)
// and ln p_j = ln 2 ((z_j - m) c - log2 S). A row whose entries all are the
// type's lowest value is a uniform one, not an overflow. A row of -inf only has
// no distribution and gives NaN.
//
// Statistics are held in fp32 per warp (a reference near the maximum, the sum,
// and for the entropy A = sum 2^x x with x = (z_j - m) c), rescaled when the
// reference grows, and joined in a fixed order, so results do not depend on
// timing.
#pragma once

#include <ATen/ATen.h>
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>
#include <map>
#include <tuple>
#include <type_traits>
#include <utility>

#include "host_utils.h"
#include "token_losses.h"

namespace kb {
namespace {  // per translation unit: each source compiles its own kernels from these

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kMaxList = kMaxTopK;

template <typename T>
struct Elem;
template <>
struct Elem<__nv_bfloat16> {
  static constexpr int kUnit = 8;
  static constexpr uint32_t kNegInf = 0xFF80FF80u;
  static __device__ __forceinline__ float load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ void store(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
  static __device__ __forceinline__ void unpack(const uint4& q, float (&v)[8]) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
  static __device__ __forceinline__ uint4 pack(const float (&v)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  // Largest of the unit's elements; NaN when there is one.
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
  }
  static __device__ __forceinline__ float widen_max(uint32_t w) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(__uint_as_float(w << 16)), "f"(__uint_as_float(w & 0xFFFF0000u)));
    return d;
  }
};
template <>
struct Elem<__half> {
  static constexpr int kUnit = 8;
  static constexpr uint32_t kNegInf = 0xFC00FC00u;
  static __device__ __forceinline__ float load(const __half* p) { return __half2float(*p); }
  static __device__ __forceinline__ void store(__half* p, float v) { *p = __float2half_rn(v); }
  static __device__ __forceinline__ void unpack(const uint4& q, float (&v)[8]) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
  static __device__ __forceinline__ uint4 pack(const float (&v)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
  }
  static __device__ __forceinline__ float widen_max(uint32_t w) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(f.x), "f"(f.y));
    return d;
  }
};
template <>
struct Elem<float> {
  static constexpr int kUnit = 4;
  static constexpr uint32_t kNegInf = 0xFF800000u;
  static __device__ __forceinline__ float load(const float* p) { return *p; }
  static __device__ __forceinline__ void store(float* p, float v) { *p = v; }
  static __device__ __forceinline__ void unpack(const uint4& q, float (&v)[4]) {
    v[0] = __uint_as_float(q.x);
    v[1] = __uint_as_float(q.y);
    v[2] = __uint_as_float(q.z);
    v[3] = __uint_as_float(q.w);
  }
  static __device__ __forceinline__ uint4 pack(const float (&v)[4]) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  }
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(__uint_as_float(a)), "f"(__uint_as_float(b)));
    return __float_as_uint(d);
  }
  static __device__ __forceinline__ float widen_max(uint32_t w) { return __uint_as_float(w); }
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// Pairs of fp32 values in one 64-bit register: one instruction per two elements.
using F2 = unsigned long long;
__device__ __forceinline__ F2 pair(float a, float b) {
  F2 d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float2 split(F2 v) {
  float2 d;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(d.x), "=f"(d.y) : "l"(v));
  return d;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}

// A row cut for 16-byte access: `head` elements before the first 16-byte
// boundary, `units` whole units, the rest behind them. The (fewer than two
// units of) elements outside whole units are the row's ragged ones.
template <typename T>
struct Row {
  const T* z;
  int head, units, ragged;
  __device__ __forceinline__ Row(const T* p, int V) : z(p) {
    constexpr int E = Elem<T>::kUnit;
    const int to_boundary = (int)(((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / sizeof(T));
    head = min(V, to_boundary);
    units = (V - head) / E;
    ragged = V - units * E;
  }
  __device__ __forceinline__ const uint4* unit_ptr() const { return reinterpret_cast<const uint4*>(z + head); }
  __device__ __forceinline__ int ragged_index(int i) const {
    return i < head ? i : units * Elem<T>::kUnit + i;
  }
};

constexpr int kBatch = 4;  // units of a thread's batch of loads

// Statistics of a set of elements: maximum, S and A (see above).
struct Acc {
  float m = -INFINITY, s = 0.f, a = 0.f;
  // Joins another set's statistics.
  template <bool ENT>
  __device__ __forceinline__ void join(float m2, float s2, float a2, float c) {
    const float mn = max_nan(m, m2);
    const float x1 = (m - mn) * c, x2 = (m2 - mn) * c;
    const float f1 = (m == mn) ? 1.f : ex2(x1), f2 = (m2 == mn) ? 1.f : ex2(x2);
    if (ENT) {
      const float y1 = (m == mn) ? 0.f : fmaxf(x1, -1e30f), y2 = (m2 == mn) ? 0.f : fmaxf(x2, -1e30f);
      a = f1 * (a + s * y1) + f2 * (a2 + s2 * y2);
    }
    s = s * f1 + s2 * f2;
    m = mn;
  }
};

__device__ __forceinline__ float warp_max_nan(float v) {
  float d;
  asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(d) : "f"(v));
  return d;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Running statistics of a warp's elements: sums of 2^x with x = z c - r, for a
// reference r that all lanes share, so that they need no rescaling when they are
// joined; each lane holds its sums as two halves. With m the largest element when
// the reference was last taken, r is m c rounded, which makes x one exact
// product and one rounding; total() makes up for the rounding of r, which is
// at most 1/2 below 2^24. Where m c is larger (a mask like -1e30, or infinite
// or NaN), r could be off by more than 2^x can hold, and x = (z - m) c instead.
template <bool ENT>
struct Run {
  float m = -INFINITY, r = 0.f;
  bool plain = false;  // x = z c - r
  F2 s{}, a{};
  // Takes the reference up to the largest of the lanes' `wide`; called by whole warps.
  __device__ __forceinline__ void raise(float wide, float c) {
    if (!__any_sync(0xffffffffu, !(wide <= m))) return;
    const float mn = max_nan(m, warp_max_nan(wide)), rn = mn * c;
    const bool pn = fabsf(rn) < 16777216.f;
    // From the old reference, r or m c, to the new one.
    const float x = plain ? (pn ? r - rn : fmaf(-mn, c, r)) : pn ? fmaf(m, c, -rn) : (m - mn) * c;
    const float f = (m == mn) ? 1.f : ex2(x);
    const F2 ff = pair(f, f);
    if (ENT) {
      const float y = fmaxf(x, -1e30f);  // the sum is 0 where x is -inf
      a = mul2(ff, fma2(s, pair(y, y), a));
    }
    s = mul2(s, ff);
    m = mn;
    r = rn;
    plain = pn;
  }
  // Two elements where `plain`.
  __device__ __forceinline__ void add(F2 z, F2 c, F2 minus_r) {
    const F2 x = fma2(z, c, minus_r);
    const float2 xs = split(x);
    const F2 e = pair(ex2(xs.x), ex2(xs.y));
    s = add2(s, e);
    if (ENT) a = fma2(e, x, a);
  }
  // An element's x in any case; -inf for a masked one.
  __device__ __forceinline__ float exponent(float z, float c) const {
    return plain ? fmaf(z, c, -r) : (z - (m == -INFINITY ? 0.f : m)) * c;
  }
  // An element in any case; with ONLY_A its part of A alone. 2^-inf (-inf) is 0.
  template <bool ONLY_A>
  __device__ __forceinline__ void add_any(float z, float c) {
    const float x = exponent(z, c), e = ex2(x);
    if (!ONLY_A) s = add2(s, pair(e, 0.f));
    if (ENT) a = fma2(pair(e, 0.f), pair(fmaxf(x, -256.f), 0.f), a);
  }
  // One element per lane (-inf for none); called by whole warps.
  __device__ __forceinline__ void add_one(float z, float c) {
    raise(z, c);
    add_any<false>(z, c);
  }
  // What every x is too large by, to the reference's m.
  __device__ __forceinline__ float offset(float c) const { return plain ? fmaf(m, c, -r) : 0.f; }
  // The warp's maximum and sum to its reference's m, in every lane.
  __device__ __forceinline__ Acc total(float c) const {
    Acc t;
    const float2 ss = split(s);
    t.m = m;
    t.s = warp_sum(ss.x + ss.y) * ex2(-offset(c));
    return t;
  }
};

__device__ __forceinline__ uint4 load_unit(const uint4* p) {
  uint4 q;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w)
               : "l"(p));
  return q;
}

// KEEP leaves the line in L2 for writes that follow; without, it may go first.
template <bool KEEP>
__device__ __forceinline__ void store_unit(uint4* p, const uint4& q) {
  if (KEEP)
    asm volatile("st.global.v4.u32 [%0], {%1, %2, %3, %4};" ::"l"(p), "r"(q.x), "r"(q.y), "r"(q.z), "r"(q.w) : "memory");
  else
    asm volatile("st.global.cs.v4.u32 [%0], {%1, %2, %3, %4};" ::"l"(p), "r"(q.x), "r"(q.y), "r"(q.z), "r"(q.w)
                 : "memory");
}

// Masks the elements of a unit whose bit is set in `b`.
template <typename T>
__device__ __forceinline__ void mask_unit(uint4& q, uint32_t b) {
  uint32_t* w = reinterpret_cast<uint32_t*>(&q);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (Elem<T>::kUnit == 8) {
      const uint32_t keep = ((b >> (2 * i)) & 1u ? 0u : 0xFFFFu) | ((b >> (2 * i + 1)) & 1u ? 0u : 0xFFFF0000u);
      w[i] = (w[i] & keep) | (Elem<T>::kNegInf & ~keep);
    } else if ((b >> i) & 1u) {
      w[i] = Elem<T>::kNegInf;
    }
  }
}

// Marks of elements of a part of a row: the bits of a thread's batch lie together (a byte per unit of eight elements,
// half a byte per unit of four), so that a thread finds with one load that none of its batch is marked. One more word is
// for the ragged elements.
template <typename T, int NT>
struct Marks {
  static constexpr int E = Elem<T>::kUnit;
  uint32_t* words;
  int u0, u1;
  __device__ __forceinline__ Marks(uint32_t* w, int first, int last) : words(w), u0(first), u1(last) {}
  static __host__ __device__ __forceinline__ int size(int units) {
    return (units + kBatch * NT - 1) / (kBatch * NT) * (NT * E / 8) + 1;
  }
  // The place of a token's bit, if it lies in this part.
  __device__ __forceinline__ bool place(const Row<T>& row, int id, bool ragged_too, int& bit) const {
    const int at = id - row.head;
    if (at < 0 || at >= row.units * E) {
      bit = (size(u1 - u0) - 1) * 32 + (at < 0 ? id : id - row.units * E);
      return ragged_too;
    }
    const int u = at / E - u0;
    bit = ((u / (kBatch * NT) * NT + u % NT) * kBatch + u / NT % kBatch) * E + at % E;
    return u >= 0 && u < u1 - u0;
  }
  // Whether it was marked before.
  __device__ __forceinline__ bool mark(const Row<T>& row, int id, bool ragged_too) const {
    int bit;
    return place(row, id, ragged_too, bit) && ((atomicOr(words + bit / 32, 1u << (bit % 32)) >> (bit % 32)) & 1u);
  }
  // Forgets all marks next to a token's.
  __device__ __forceinline__ void unmark(const Row<T>& row, int id) const {
    int bit;
    if (place(row, id, true, bit)) words[bit / 32] = 0;
  }
  __device__ __forceinline__ bool ragged(int i) const { return (words[size(u1 - u0) - 1] >> i) & 1u; }
  __device__ __forceinline__ uint32_t of_batch(int batch) const {
    const int at = batch * NT + threadIdx.x;
    return E == 8 ? words[at] : reinterpret_cast<const uint16_t*>(words)[at];
  }
};
struct NoMarks {};

// Where a row's units come from: memory, or units [u0, ..) staged in shared memory.
struct FromMemory {
  static constexpr bool kPatch = false;
  const uint4* p;
  __device__ __forceinline__ void begin(int) const {}
  __device__ __forceinline__ uint4 load(int u) const { return load_unit(p + u); }
};

// Statistics of the units [u0, u1) of a row over the threads of a block, in
// batches of four 16-byte loads per thread (unit u0 + tid + (4 b + i) NT is the
// i-th of batch b). With MAX, batch_max(b, m) gets each batch's maximum, and the
// reference follows it. Without, the first batch gives the reference, and a
// later one is taken again with a new one only if its sum has grown past
// 2^20 (the maximum is at most 20 off then, which costs the entropy 20 2^-23):
// half an instruction per element less. Per element that leaves the widening,
// and in pairs a multiply-add, two 2^x and one or two sums.
// Clamping masked entries' exponents would cost one more instruction per
// element; instead a batch whose A came out NaN (0 times -inf) takes its A again.
template <typename T, int NT, bool MAX, bool ENT, typename Src, typename M, typename G>
__device__ __forceinline__ void stream_units(const Src& src, int u0, int u1, float c, Run<ENT>& run, const M& marks,
                                             const G& batch_max) {
  constexpr bool MASK = !std::is_same_v<M, NoMarks>;
  static_assert(!(ENT && MASK), "the masked form takes no entropy");
  constexpr int UN = kBatch, E = Elem<T>::kUnit;
  const F2 cc = pair(c, c);
  int batch = 0;
  for (int base = u0 + (int)(threadIdx.x & ~31u); base < u1; base += UN * NT, ++batch) {  // whole warps
    const int u = base + (int)(threadIdx.x & 31);
    const bool whole = base + (UN - 1) * NT + 32 <= u1;
    src.begin(batch);
    uint32_t set = 0;
    if constexpr (MASK) {
      set = marks.of_batch(batch);
      if constexpr (Src::kPatch) {
        // The lane's own units: no one else reads them.
        for (; set; set &= set - 1) {
          const int b = __ffs(set) - 1;
          src.template patch<T>(u + b / E * NT, b % E);
        }
      }
    }
    uint4 q[UN];
    if (whole) {
#pragma unroll
      for (int i = 0; i < UN; ++i) q[i] = src.load(u + i * NT);
    } else {
#pragma unroll
      for (int i = 0; i < UN; ++i) {
        q[i] = make_uint4(Elem<T>::kNegInf, Elem<T>::kNegInf, Elem<T>::kNegInf, Elem<T>::kNegInf);
        if (u + i * NT < u1) q[i] = src.load(u + i * NT);
      }
    }
    if constexpr (MASK) {
      if (set) {
#pragma unroll
        for (int i = 0; i < UN; ++i)
          if ((set >> (E * i)) & ((1u << E) - 1u)) mask_unit<T>(q[i], set >> (E * i));
      }
    }
    if (MAX || run.m == -INFINITY) {
      uint32_t mx = Elem<T>::max2(Elem<T>::max2(q[0].x, q[0].y), Elem<T>::max2(q[0].z, q[0].w));
#pragma unroll
      for (int i = 1; i < UN; ++i)
        mx = Elem<T>::max2(mx, Elem<T>::max2(Elem<T>::max2(q[i].x, q[i].y), Elem<T>::max2(q[i].z, q[i].w)));
      const float wide = Elem<T>::widen_max(mx);
      batch_max(batch, wide);
      run.raise(wide, c);
    }
    const F2 s_before = run.s, a_before = run.a;
    bool again = !run.plain;
    if (run.plain) {
      const F2 rr = pair(-run.r, -run.r);
#pragma unroll
      for (int i = 0; i < UN; ++i) {
        if (whole || base + i * NT < u1) {  // lanes behind the end hold -inf
          float v[E];
          Elem<T>::unpack(q[i], v);
#pragma unroll
          for (int j = 0; j < E; j += 2) run.add(pair(v[j], v[j + 1]), cc, rr);
        }
      }
      if (!MAX) {
        const float2 ss = split(run.s);
        again = __any_sync(0xffffffffu, !(ss.x + ss.y <= 1048576.f));
      }
    }
    // The ways below are rare and read the batch again.
    if (again) {
      run.s = s_before;
      run.a = a_before;
      for (int pass = MAX ? 1 : 0; pass < 2; ++pass) {
        float wide = -INFINITY;
#pragma unroll 1
        for (int i = 0; i < UN; ++i) {
          if (u + i * NT >= u1) continue;
          uint4 w = src.load(u + i * NT);
          if (MASK) mask_unit<T>(w, set >> (E * i));
          float v[E];
          Elem<T>::unpack(w, v);
#pragma unroll
          for (int j = 0; j < E; ++j) {
            if (pass == 0) wide = max_nan(wide, v[j]);
            else run.template add_any<false>(v[j], c);
          }
        }
        if (pass == 0) run.raise(wide, c);
      }
    } else if (ENT) {
      const float2 aa = split(run.a);
      if (!(aa.x + aa.y == aa.x + aa.y)) {
        run.a = a_before;
#pragma unroll 1
        for (int i = 0; i < UN; ++i) {
          if (u + i * NT >= u1) continue;
          float v[E];
          Elem<T>::unpack(src.load(u + i * NT), v);
#pragma unroll
          for (int j = 0; j < E; ++j) run.template add_any<true>(v[j], c);
        }
      }
    }
  }
}

// Joins statistics held by the first N lanes of a warp (N a power of two); every lane returns with them.
template <int N, bool ENT>
__device__ __forceinline__ Acc join_lanes(Acc v, float c) {
  Acc r;
  const bool mine = (int)(threadIdx.x & 31) < N;
  r.m = warp_max_nan(mine ? v.m : -INFINITY);
  const float x = (v.m - r.m) * c, f = v.m == r.m ? 1.f : ex2(x);
  float s = mine ? v.s * f : 0.f, a = 0.f;
  if (ENT) a = mine ? f * (v.a + v.s * (v.m == r.m ? 0.f : fmaxf(x, -1e30f))) : 0.f;
#pragma unroll
  for (int o = N / 2; o > 0; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    if (ENT) a += __shfl_xor_sync(0xffffffffu, a, o);
  }
  r.s = __shfl_sync(0xffffffffu, s, 0);
  r.a = ENT ? __shfl_sync(0xffffffffu, a, 0) : 0.f;
  return r;
}

// Joins the maxima and sums of a block's warps; the first warp returns with them.
template <int NT>
__device__ __forceinline__ Acc block_join(const Run<false>& run, float c, Acc* sm) {
  const Acc w = run.total(c);
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = w;
  __syncthreads();
  Acc r;
  if (threadIdx.x < 32) r = join_lanes<NT / 32, false>(sm[threadIdx.x & (NT / 32 - 1)], c);
  return r;
}

// Units of part `i` of `n`; the first part also takes the ragged elements.
__device__ __forceinline__ void segment(int units, int i, int n, int& u0, int& u1) {
  const int per = (units + n - 1) / n;
  u0 = min(units, i * per);
  u1 = min(units, u0 + per);
}

// Writes a thread's batch of units u, u + NT, ...: out = f(two elements, the index of the first). `loaded` is called
// once the batch is in registers. WHOLE: no unit of the batch is behind the end.
template <typename T, int NT, bool KEEP, bool WHOLE, typename Src, typename F, typename L>
__device__ __forceinline__ void map_batch(const Row<T>& row, const Src& src, T* out, bool same, int u, int u1,
                                          const F& f, const L& loaded) {
  constexpr int E = Elem<T>::kUnit;
  uint4 q[kBatch];
#pragma unroll
  for (int i = 0; i < kBatch; ++i)
    if (WHOLE || u + i * NT < u1) q[i] = src.load(u + i * NT);
  loaded();
#pragma unroll
  for (int i = 0; i < kBatch; ++i) {
    if (WHOLE || u + i * NT < u1) {
      const int idx = row.head + (u + i * NT) * E;
      float v[E];
      Elem<T>::unpack(q[i], v);
#pragma unroll
      for (int j = 0; j < E; j += 2) {
        const float2 d = split(f(pair(v[j], v[j + 1]), idx + j));
        v[j] = d.x;
        v[j + 1] = d.y;
      }
      if (same) {
        store_unit<KEEP>(reinterpret_cast<uint4*>(out + idx), Elem<T>::pack(v));
      } else {
#pragma unroll
        for (int j = 0; j < E; ++j) Elem<T>::store(out + idx + j, v[j]);
      }
    }
  }
}

// Whether a row and its gradient lie alike to 16-byte boundaries.
template <typename T>
__device__ __forceinline__ bool same_boundaries(const T* z, const T* out) {
  return ((reinterpret_cast<uintptr_t>(z) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;
}

// The same for the units [u0, u1) of a row and, for the first segment, its ragged elements.
template <typename T, int NT, bool KEEP, typename F>
__device__ __forceinline__ void map_row(const Row<T>& row, T* out, int u0, int u1, int ragged, const F& f) {
  const bool same = same_boundaries(row.z, out);
  if ((int)threadIdx.x < ragged) {
    const int idx = row.ragged_index(threadIdx.x);
    Elem<T>::store(out + idx, split(f(pair(Elem<T>::load(row.z + idx), 0.f), idx)).x);
  }
  const FromMemory src{row.unit_ptr()};
  int u = u0 + (int)threadIdx.x;
  for (; u + (kBatch - 1) * NT < u1; u += kBatch * NT)
    map_batch<T, NT, KEEP, true>(row, src, out, same, u, u1, f, [] {});
  if (u < u1) map_batch<T, NT, KEEP, false>(row, src, out, same, u, u1, f, [] {});
}

template <typename T, int NT>
__device__ __forceinline__ void zero_row(const Row<T>& out, int u0, int u1, int ragged) {
  T* o = const_cast<T*>(out.z);
  if ((int)threadIdx.x < ragged) Elem<T>::store(o + out.ragged_index(threadIdx.x), 0.f);
  uint4* p = const_cast<uint4*>(out.unit_ptr());
  for (int u = u0 + (int)threadIdx.x; u < u1; u += NT) store_unit<false>(p + u, make_uint4(0, 0, 0, 0));
}

// ------------------------------------------------------------------ host

template <typename T>
struct Tag {
  using type = T;
};

template <typename F>
void for_logits_type(at::ScalarType dtype, F&& f) {
  switch (dtype) {
    case at::kBFloat16: f(Tag<__nv_bfloat16>{}); break;
    case at::kHalf: f(Tag<__half>{}); break;
    case at::kFloat: f(Tag<float>{}); break;
    default: KB_CHECK(false, "logits must be bf16, fp16 or fp32");
  }
}

void check_rows(const at::Tensor& t, const char* name, int64_t rows, int64_t cols, at::ScalarType dtype,
                const at::Tensor& like) {
  const std::string n(name);
  KB_CHECK(t.is_cuda() && t.device() == like.device(), n + " must be on the logits' device");
  KB_CHECK(t.scalar_type() == dtype, n + " has the wrong dtype");
  KB_CHECK(t.is_contiguous() && t.numel() == rows * cols, n + " must be contiguous with one entry per row and column");
}

// A row gradient: fp32, one per row, contiguous (stride 1) or expanded from one value (stride 0).
struct RowGrad {
  const float* p;
  int stride;
  __device__ __forceinline__ float at(long long row, float none) const { return p ? p[row * stride] : none; }
};
RowGrad check_row_grad(const c10::optional<at::Tensor>& t, const char* name, int64_t rows, const at::Tensor& like) {
  if (!t) return RowGrad{nullptr, 0};
  const std::string n(name);
  KB_CHECK(t->is_cuda() && t->device() == like.device() && t->scalar_type() == at::kFloat, n + " must be fp32 on the logits' device");
  KB_CHECK(t->dim() == 1 && t->size(0) == rows && (rows <= 1 || t->stride(0) == 1 || t->stride(0) == 0),
           n + " must hold one value per row, contiguous or expanded");
  return RowGrad{t->data_ptr<float>(), rows <= 1 || t->stride(0) == 0 ? 0 : 1};
}

// logits [rows, >= vocab] with unit inner stride; returns the row count.
int64_t check_logits(const at::Tensor& logits, int64_t vocab, double temperature, const char* name) {
  const std::string n(name);
  check_cuda_tensor(logits, name);
  KB_CHECK(logits.dim() == 2, n + " must be [rows, vocab]");
  KB_CHECK(vocab >= 1 && vocab <= logits.size(1), n + " has fewer columns than the vocabulary");
  KB_CHECK(vocab <= kMaxListVocab, "vocabularies of more than 524288 entries are not supported");
  KB_CHECK(logits.size(1) == 1 || logits.stride(1) == 1, n + " must have unit inner stride");
  KB_CHECK(logits.size(0) <= 0x7FFFFFFF / 16, n + " has too many rows");
  KB_CHECK(reinterpret_cast<uintptr_t>(logits.data_ptr()) % logits.element_size() == 0, n + " is misaligned");
  KB_CHECK(temperature >= 1e-4 && temperature <= 1e4, "temperature must lie in [1e-4, 1e4]");
  return logits.size(0);
}

void check_out(const at::Tensor& out, const at::Tensor& logits, int64_t vocab) {
  KB_CHECK(out.is_cuda() && out.device() == logits.device() && out.scalar_type() == logits.scalar_type(),
           "out must have the logits' device and dtype");
  KB_CHECK(out.dim() == 2 && out.size(0) == logits.size(0) && out.size(1) >= vocab, "out must be [rows, vocab]");
  KB_CHECK(out.size(1) == 1 || out.stride(1) == 1, "out must have unit inner stride");
  KB_CHECK(out.size(0) <= 1 || out.stride(0) >= vocab, "rows of out overlap");
  // The logits themselves, or memory apart from theirs: a shifted view would be overwritten before it is read.
  if (out.numel() == 0 || out.data_ptr() == logits.data_ptr()) {
    KB_CHECK(out.numel() == 0 || out.size(0) <= 1 || out.stride(0) == logits.stride(0), "out overlaps the logits");
    return;
  }
  const auto bytes_end = [vocab](const at::Tensor& t) {
    return (const char*)t.data_ptr() + ((t.size(0) - 1) * t.stride(0) + vocab) * t.element_size();
  };
  const bool apart = bytes_end(out) <= (const char*)logits.data_ptr() || bytes_end(logits) <= (const char*)out.data_ptr();
  // Two column ranges of one buffer interleave without meeting.
  const int64_t row = out.stride(0) * out.element_size();
  const int64_t gap = ((const char*)out.data_ptr() - (const char*)logits.data_ptr()) % std::max<int64_t>(row, 1);
  const int64_t shift = gap < 0 ? gap + row : gap, width = vocab * out.element_size();
  KB_CHECK(apart || (out.stride(0) == logits.stride(0) && shift >= width && row - shift >= width),
           "out overlaps the logits");
}

// Threads per row of the statistics' passes, and blocks where a cluster shares a row. Many rows: small blocks leave less
// of the device idle at a row's end (V = 50257 bf16, 16384 rows: 264 us with 128 threads, 282 with 256, 337 with 512),
// but rows above 128 KB take 256 (V = 131072 fp32, 4096 rows: 313 against 333 us). Few rows: larger blocks (257 rows of
// 50257 bf16: 8.0 us with 512 threads, 8.4 with 256, 11.0 with 128; rows of 16 KB: 3.7 with 256, 3.9 with 512), and
// clusters while each block keeps at least 16 KB and has an SM of its own, or at least 64 KB and a third of one (one row
// of 50257 bf16: 5.1 us with four blocks, 5.8 with one; 40 rows of 131072 fp32: 6.8 with eight, 12.3 with one; but 257
// rows of 50257 bf16: 9.7 with two, 8.0 with one). A `light` kernel, of which an SM holds three blocks of 512 threads or
// five of 256, takes long rows by waves: 512 threads up to three rows per SM, which all run at once then, 256 up to five
// and a little more, 512 up to nine, where three whole waves beat one and a part of a second (distillation, rows of
// 131072 fp32, 512 against 256 threads in us: 400 rows 36 and 42, 700 62 and 58, 850 71 and 69, 1024 91 and 102, 1200 99
// and 108, 1500 124 and 120, 2048 161 and 168, 4096 314 and 305; of 50257 fp32: 400 15 and 18, 700 27 and 23, 850 31 and
// 28, 1024 39 and 42, 1200 43 and 44, 1500 54 and 48). Log probabilities, of which an SM holds two blocks of 512 threads,
// take 256 (rows of 131072 fp32: 1024 rows 89 and 90 us, 700 65 and 55).
struct RowLaunch {
  int threads, parts;
};
RowLaunch row_launch(int64_t rows, int64_t row_bytes, bool light, int device) {
  const int64_t sms = num_sms(device);
  RowLaunch how{128, 1};
  while (how.parts < 8) {
    const int64_t blocks = rows * how.parts * 2, part = row_bytes / (how.parts * 2);
    if (!(part >= 16384 && blocks <= sms) && !(part >= 65536 && blocks <= 3 * sms)) break;
    how.parts *= 2;
  }
  if (how.parts > 1) how.threads = 256;
  else if (row_bytes <= 32768) how.threads = rows < 400 && row_bytes >= 8192 ? 256 : 128;
  else if (rows <= 2 * sms) how.threads = 512;
  else if (row_bytes > 131072 && light && (rows <= 3 * sms || (rows > 6 * sms && rows <= 9 * sms))) how.threads = 512;
  else if (rows < 1000 || row_bytes > 131072) how.threads = 256;
  return how;
}

template <int N>
using Int = std::integral_constant<int, N>;
template <typename F>
void for_bool(bool b, F&& f) {
  if (b) f(std::true_type{});
  else f(std::false_type{});
}
template <typename F>
void for_row_launch(const RowLaunch& how, F&& f) {
  if (how.parts > 1) f(Int<256>{}, std::true_type{});
  else if (how.threads == 128) f(Int<128>{}, std::false_type{});
  else if (how.threads == 256) f(Int<256>{}, std::false_type{});
  else f(Int<512>{}, std::false_type{});
}

// Lets a kernel use `smem` bytes of dynamic shared memory; with `threads`, returns how many of its blocks an SM holds.
// The limit is one value per kernel and device, which calls with other sizes share: it is only ever raised.
template <typename Kern>
int allow_smem(Kern kern, size_t smem, int threads, int device) {
  static std::mutex mu;
  static std::map<std::pair<const void*, int>, size_t> limits;
  static std::map<std::tuple<const void*, int, size_t, int>, int> known;
  const void* const id = reinterpret_cast<const void*>(kern);
  std::lock_guard<std::mutex> lock(mu);
  size_t& limit = limits.try_emplace({id, device}, 32 * 1024).first->second;
  if (smem > limit) {
    KB_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    limit = smem;
  }
  if (!threads) return 0;
  const auto at = known.try_emplace({id, device, smem, threads}, 0);
  if (at.second)
    KB_CUDA_CHECK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&at.first->second, kern, threads, smem));
  return at.first->second;
}

template <typename... P, typename... A>
void launch_rows(void (*kern)(P...), int64_t rows, int threads, int parts, size_t smem, cudaStream_t s, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * parts));
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)parts;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = parts > 1 ? 1 : 0;
  KB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, static_cast<P>(args)...));
}

// Rows of a gradient up to here are written by 64 threads: more have nothing to do.
constexpr int64_t kSmallRow = 8192;

int row_segments(int64_t rows, int64_t vocab, int64_t elem, int threads, int device) {
  const int64_t units = vocab * elem / 16;
  const int64_t most = std::max<int64_t>(1, units / (2 * threads));
  const int64_t want = (4 * (int64_t)num_sms(device) + rows - 1) / rows;
  return (int)std::max<int64_t>(1, std::min<int64_t>({most, want, 64}));
}

}  // namespace
}  // namespace kb
