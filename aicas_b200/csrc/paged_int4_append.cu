// Append to and reads from a paged KV cache of 4-bit rows.
//
//   y = x * rsqrt(mean x^2 + eps) * w        (with a norm weight, else y = x)
//   r = y * cos + rotate_half(y) * sin,      rotate_half(y) = cat(-y[D/2:], y[:D/2])
//   of each group of 64 (or D) elements of r (keys) and v:
//     least = T(min r),  scale = T((max r - least) * (1 / 15)), an fp32 product with fp32's 1 / 15
//     code  = (r - least) / scale to the nearest of 0..15   (0 where scale is no normal fp32 number)
//   read back as fma(scale, code, least), rounded to T.
//
// Rounding of r: paged_append.cu's (fp32 tables: fp32 to the code; 16-bit tables: every
// operation).  The codes are taken against the rounded least and scale, so that what
// rounding those two moved is not added to a code's own half step.
#include <cstdio>
#include <type_traits>

#include "common.cuh"
#include "paged_int4.cuh"
#include "paged_rows.cuh"

namespace aicas {
namespace {

// Least and largest of three; NaN if one is.
__device__ __forceinline__ float min_nan(float a, float b, float c) {
  float r;
  asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// And of 8 elements.
__device__ __forceinline__ void range8(const float* x, float& lo, float& hi) {
  lo = min_nan(min_nan(x[0], x[1], x[2]), min_nan(x[3], x[4], x[5]), min_nan(x[6], x[7], x[7]));
  hi = max_nan(max_nan(x[0], x[1], x[2]), max_nan(x[3], x[4], x[5]), max_nan(x[6], x[7], x[7]));
}

// Least and largest of a group over its TPR lanes; NaN where an element is.
template <int TPR>
__device__ __forceinline__ void group_range(uint32_t lanes, float& lo, float& hi) {
#pragma unroll
  for (int off = TPR / 2; off >= 1; off >>= 1) {
    lo = min_nan(lo, lo, __shfl_xor_sync(lanes, lo, off));
    hi = max_nan(hi, hi, __shfl_xor_sync(lanes, hi, off));
  }
}

// Two numbers, two operations an instruction (8 prompts of 2048 tokens written and read back 80 ->
// 78 us).  The assembler may fuse a product that is added to something, .rn or not: where both
// roundings are wanted it takes the operations of single numbers.
struct Two {
  uint64_t u;
  Two() = default;
  __device__ __forceinline__ Two(float x, float y) { asm("mov.b64 %0, {%1, %2};" : "=l"(u) : "f"(x), "f"(y)); }
  __device__ __forceinline__ explicit Two(float x) : Two(x, x) {}
  __device__ __forceinline__ void get(float& x, float& y) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(u)); }
};
__device__ __forceinline__ Two operator+(Two a, Two b) {
  asm("add.rn.f32x2 %0, %0, %1;" : "+l"(a.u) : "l"(b.u));
  return a;
}
__device__ __forceinline__ Two operator*(Two a, Two b) {
  asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(a.u) : "l"(b.u));
  return a;
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(c.u) : "l"(a.u), "l"(b.u));
  return c;
}

// A group's (scale, least) as the cache holds them, and what its codes are taken by.
struct Levels {
  float scale, least, inv;
  uint32_t pair;

  template <typename T>
  __device__ __forceinline__ void set(float lo, float hi) {
    const T l = Elem<T>::from_float(lo);
    least = Elem<T>::to_float(l);
    const T s = Elem<T>::from_float((hi - least) * (1.f / 15.f));
    scale = Elem<T>::to_float(s);
    if (!(fabsf(scale) < INFINITY)) scale = least = __int_as_float(0x7fc00000);  // an infinity or NaN among the elements
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(scale));
    inv = scale >= 0x1p-126f ? inv : 0.f;
    union {
      T t[2];
      uint32_t u;
    } r;
    r.t[0] = Elem<T>::from_float(scale), r.t[1] = Elem<T>::from_float(least);
    pair = r.u;
  }

  // The codes of 8 elements, 4 bits each.  The quotient by the reciprocal may fall on the
  // other side of a border between two codes, on which 16-bit values often lie: what a
  // nearby code leaves, which fma gives exactly, corrects it.
  __device__ __forceinline__ uint32_t codes(const float* x) const {
    if (inv == 0.f) return 0u;  // one value, or NaN
    // 1.5 x 2^23: a sum with it has the number, rounded to a whole one, in its low bits
    constexpr float kWhole = 12582912.f;
    const Two at(fmaf(-least, inv, kWhole)), by(inv), down(-scale), from(-least);
    uint32_t u = 0;
#pragma unroll
    for (int i = 6; i >= 0; i -= 2) {
      const Two v(x[i], x[i + 1]), near = fma2(v, by, at) + Two(-kWhole);
      // as so many of the smallest steps: the number, rounded to a whole one
      const Two w = fma2(fma2(near, down, v + from), by, near) * Two(0x1p-149f);
      float a, b;
      w.get(a, b);
      // two numbers, held to 0..15, below what is there
      asm("cvt.pack.sat.u4.s32.b32 %0, %1, %2, %0;" : "+r"(u) : "r"(__float_as_int(b)), "r"(__float_as_int(a)));
    }
    return u;
  }
};

// The sum of a row's squares, added in the order of torch's sums of 64 and 128 contiguous
// numbers on the GPU: x1, x2 are 8 elements each of the row's halves.
template <int D>
__device__ __forceinline__ float torch_sum(uint32_t lanes, const float* x1, const float* x2) {
  if constexpr (D == 128) {  // fours one after the other; then the halves of the 32 sums, of those, and so on
    float a[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float s[2];
#pragma unroll
      for (int side = 0; side < 2; ++side) {
        const float* x = (side == 0 ? x1 : x2) + 4 * h;
        s[side] = __fadd_rn(__fadd_rn(__fadd_rn(__fmul_rn(x[0], x[0]), __fmul_rn(x[1], x[1])), __fmul_rn(x[2], x[2])), __fmul_rn(x[3], x[3]));
      }
      a[h] = s[0] + s[1];
#pragma unroll
      for (int off = 4; off >= 1; off >>= 1) a[h] += __shfl_xor_sync(lanes, a[h], off);
    }
    return a[0] + a[1];
  } else {  // the halves of the 64 squares, of their sums, and so on
    float a[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      a[i] = __fadd_rn(__fmul_rn(x1[i], x1[i]), __fmul_rn(x2[i], x2[i]));
#pragma unroll
      for (int off = 2; off >= 1; off >>= 1) a[i] += __shfl_xor_sync(lanes, a[i], off);
    }
    return ((a[0] + a[4]) + (a[2] + a[6])) + ((a[1] + a[5]) + (a[3] + a[7]));
  }
}

// The lane's part of one token: c is its place in a row's halves, lanes those of its row.
template <typename CS, int D>
struct Token {
  static constexpr int kV = 8, kTpr = D / (2 * kV);
  int b, s, c;
  uint32_t lanes;
  int page, row;  // page -1: nowhere to write
  float c1[kV], c2[kV], s1[kV], s2[kV];  // s1 negated where tables are wider than T
};

// Where row 0 of token s of request b is, of q (kind 0), k (1) or v (2), and how far the next one.
template <typename T>
__device__ __forceinline__ const T* row_source(const aicas_paged_append_int4_params& a, int kind, int b, int s, int64_t& step) {
  step = kind == 0 ? a.qi_stride_h : kind == 1 ? a.k_stride_h : a.v_stride_h;
  return static_cast<const T*>(kind == 0 ? a.q_in : kind == 1 ? a.k_in : a.v_in) +
         b * (kind == 0 ? a.qi_stride_b : kind == 1 ? a.k_stride_b : a.v_stride_b) +
         s * (kind == 0 ? a.qi_stride_s : kind == 1 ? a.k_stride_s : a.v_stride_s);
}

// Rows h, h + step, ... (COUNT of them, below `heads`) of the token's q (KIND 0), k (1) or v (2);
// u1, u2: the lane's vectors of them.
template <typename T, typename CS, int D, bool HALVES, int KIND, int COUNT>
__device__ __forceinline__ void token_rows(const aicas_paged_append_int4_params& a, const Token<CS, D>& t, int h, int step, int heads,
                                           const uint4 (&u1)[COUNT], const uint4 (&u2)[COUNT]) {
  using K = Token<CS, D>;
  constexpr int kV = K::kV, kTpr = K::kTpr;
  constexpr bool kRoundEach = std::is_same<T, CS>::value;
  // Keys in fp32: every operation rounded as torch's, so that they get the codes that torch's keys
  // would get (a fused product and sum puts some on the other side of a border).
  constexpr bool kAsTorch = KIND == 1 && !kRoundEach;
  const T* w = static_cast<const T*>(KIND == 0 ? a.q_norm_weight : a.k_norm_weight);
  uint4 w1 = {}, w2 = {};
  if (KIND < 2 && w != nullptr) {
    w1 = *reinterpret_cast<const uint4*>(w + t.c);
    w2 = *reinterpret_cast<const uint4*>(w + t.c + D / 2);
  }
#pragma unroll
  for (int j = 0; j < COUNT; ++j) {
    const int head = h + j * step;
    if (head >= heads || (KIND > 0 && t.page < 0)) continue;  // the lanes of a row stay together
    float x1[kV], x2[kV];
    Elem<T>::unpack(u1[j], x1);
    Elem<T>::unpack(u2[j], x2);
    if constexpr (KIND < 2) {
      if (w != nullptr) {
        float f1[kV], f2[kV];
        Elem<T>::unpack(w1, f1);
        Elem<T>::unpack(w2, f2);
        float ss = 0.f;
        if constexpr (kAsTorch) {
          ss = torch_sum<D>(t.lanes, x1, x2);
        } else {
#pragma unroll
          for (int i = 0; i < kV; ++i) ss += x1[i] * x1[i] + x2[i] * x2[i];
#pragma unroll
          for (int off = kTpr / 2; off >= 1; off >>= 1) ss += __shfl_xor_sync(t.lanes, ss, off);
        }
        const float inv = rsqrtf(ss / (float)D + a.norm_eps);
        if constexpr (kAsTorch) {
#pragma unroll
          for (int i = 0; i < kV; ++i) {
            x1[i] = __fmul_rn(__fmul_rn(x1[i], inv), f1[i]);
            x2[i] = __fmul_rn(__fmul_rn(x2[i], inv), f2[i]);
          }
        } else if constexpr (kRoundEach) {
          normed_pair<T, true, kV>(x1, x2, f1, f2, inv);
        } else {
#pragma unroll
          for (int i = 0; i < kV; i += 2) {
            (Two(x1[i], x1[i + 1]) * (Two(inv) * Two(f1[i], f1[i + 1]))).get(x1[i], x1[i + 1]);
            (Two(x2[i], x2[i + 1]) * (Two(inv) * Two(f2[i], f2[i + 1]))).get(x2[i], x2[i + 1]);
          }
        }
      }
      if constexpr (kRoundEach) {
        rotated_pair<T, true, kV>(x1, x2, t.c1, t.c2, t.s1, t.s2);
      } else if constexpr (kAsTorch) {
#pragma unroll
        for (int i = 0; i < kV; ++i) {
          const float p1 = x1[i], p2 = x2[i];
          x1[i] = __fadd_rn(__fmul_rn(p1, t.c1[i]), __fmul_rn(p2, t.s1[i]));
          x2[i] = __fadd_rn(__fmul_rn(p2, t.c2[i]), __fmul_rn(p1, t.s2[i]));
        }
      } else {
#pragma unroll
        for (int i = 0; i < kV; i += 2) {
          const Two p1(x1[i], x1[i + 1]), p2(x2[i], x2[i + 1]);
          const Two c1(t.c1[i], t.c1[i + 1]), c2(t.c2[i], t.c2[i + 1]), m1(t.s1[i], t.s1[i + 1]), s2(t.s2[i], t.s2[i + 1]);
          fma2(p1, c1, p2 * m1).get(x1[i], x1[i + 1]);
          fma2(p2, c2, p1 * s2).get(x2[i], x2[i + 1]);
        }
      }
    }
    if constexpr (KIND == 0) {
      T* dst = static_cast<T*>(a.q_out) + t.b * a.qo_stride_b + t.s * a.qo_stride_s + head * a.qo_stride_h + t.c;
      *reinterpret_cast<uint4*>(dst) = pack_vec<T>(x1);
      *reinterpret_cast<uint4*>(dst + D / 2) = pack_vec<T>(x2);
    } else {
      if constexpr (KIND == 1 && kRoundEach) {
#pragma unroll
        for (int i = 0; i < kV; ++i) x1[i] = rounded<T>(x1[i]), x2[i] = rounded<T>(x2[i]);
      }
      const aicas_int4_pages& to = a.kv[KIND - 1];
      uint8_t* codes = static_cast<uint8_t*>(to.codes) + t.page * to.cs_p + t.row * to.cs_t + head * to.cs_h + t.c / 2;
      T* pair = static_cast<T*>(to.scales) + t.page * to.ss_p + t.row * to.ss_t + head * to.ss_h;
      float lo1, hi1, lo2, hi2;
      range8(x1, lo1, hi1);
      range8(x2, lo2, hi2);
      Levels v1 = {}, v2 = {};
      if constexpr (HALVES) {
        group_range<kTpr>(t.lanes, lo1, hi1);
        group_range<kTpr>(t.lanes, lo2, hi2);
        v1.set<T>(lo1, hi1);
        v2.set<T>(lo2, hi2);
        if (t.c == 0) *reinterpret_cast<uint2*>(pair) = make_uint2(v1.pair, v2.pair);
      } else {
        lo1 = min_nan(lo1, lo1, lo2), hi1 = max_nan(hi1, hi1, hi2);
        group_range<kTpr>(t.lanes, lo1, hi1);
        v1.set<T>(lo1, hi1);
        v2 = v1;
        if (t.c == 0) *reinterpret_cast<uint32_t*>(pair) = v1.pair;
      }
      *reinterpret_cast<uint32_t*>(codes) = v1.codes(x1);
      *reinterpret_cast<uint32_t*>(codes + D / 4) = v2.codes(x2);
    }
  }
}

// The token's rows are read once, q is written in 16 and k and v in 4 bits.  As in
// paged_append.cu a row (one head of q, k or v) belongs to D / 16 threads, each with one
// 16-byte vector of the row's first half and the matching one of its second half, so that the
// rotation needs no exchange, and with groups of 64 in rows of 128 each half is a group.
// PROMPT: a warp walks through tokens, a unit of two rows a lane at a time; the units are
// copied into shared memory kUnits ahead, and the next token's tables, each lane's vectors by
// itself, so that the lanes wait for no one.  Else a CTA a token, a row a thread, all at once.
//
// One token of 16 query and 8 KV heads of 128 and its read back 4.0 us, 64 tokens 4.3: two
// launches.  8 prompts of 2048 tokens and their read back 72 us, 4.2 TB/s: about 2200
// instructions a token, whose chains 16 warps an SM (of 128 registers a thread) cover to 63% of
// the issue slots, while the memory is at 44%.  Without the copies ahead 78 us; rows asked for
// ahead in registers 92, 20 and 24 warps an SM 79 and 104.
constexpr int kPromptWarps = 4, kPromptCtas = 4;  // of a CTA, of an SM
constexpr int kUnits = 2;  // 8 prompts of 2048 tokens with 2 74.0 us, 4 74.8, 6 76.8

// A token's page (-1: nowhere to write) and row in it; its request's length, where one is asked for.
__device__ __forceinline__ int2 place_of(const aicas_paged_append_int4_params& a, int b, int s, bool first_lane) {
  const int pos = a.positions[b];
  const int fresh = a.num_new != nullptr ? min(max(a.num_new[b], 0), a.seq_len) : a.seq_len;
  const int cap = a.max_pages * a.page_size;
  const long long slot = (long long)pos + s;
  int2 at = make_int2(-1, 0);
  if (s < fresh && slot >= 0 && slot < cap) {
    const int i = (int)((uint32_t)slot / (uint32_t)a.page_size);
    at = make_int2(a.page_table[b * a.table_stride + i], (int)slot - i * a.page_size);
    if (at.x >= a.num_pages) at.x = -1;
  }
  if (a.kv_lens_out != nullptr && s == 0 && first_lane) a.kv_lens_out[b] = (int)min((long long)max(pos, 0) + fresh, (long long)cap);
  return at;
}

// cos and sin of a token's dims c .. c + 7 and D / 2 + c .. as the rotation takes them, from the four places.
template <typename T, typename CS, int D>
__device__ __forceinline__ void take_tables(Token<CS, D>& t, const CS* c1, const CS* c2, const CS* s1, const CS* s2) {
  constexpr int kV = Token<CS, D>::kV;
  load_floats<CS, kV>(c1, t.c1);
  load_floats<CS, kV>(c2, t.c2);
  load_floats<CS, kV>(s1, t.s1);
  load_floats<CS, kV>(s2, t.s2);
  if constexpr (!std::is_same<T, CS>::value)
#pragma unroll
    for (int i = 0; i < kV; ++i) t.s1[i] = -t.s1[i];
}

template <typename T, typename CS, int D, bool HALVES>
__global__ void __launch_bounds__(256, 1) paged_append_int4_kernel(const __grid_constant__ aicas_paged_append_int4_params a) {
  using K = Token<CS, D>;
  constexpr int kTpr = K::kTpr, kSlots = 256 / kTpr;
  K t;
  t.c = threadIdx.x % kTpr * K::kV;
  t.lanes = ((1u << kTpr) - 1u) << (threadIdx.x % 32 / kTpr * kTpr);
  const int hq = a.num_q_heads, hkv = a.num_kv_heads;
  grid_launch_dependents();
  grid_dependency_wait();
  t.b = (int)blockIdx.x / a.seq_len, t.s = (int)blockIdx.x - t.b * a.seq_len;
  const int2 place = place_of(a, t.b, t.s, threadIdx.x == 0);  // asked for first, needed last
  t.page = place.x, t.row = place.y;
  const CS* cp = static_cast<const CS*>(a.cos) + t.b * a.cs_stride_b + t.s * a.cs_stride_s + t.c;
  const CS* sp = static_cast<const CS*>(a.sin) + t.b * a.cs_stride_b + t.s * a.cs_stride_s + t.c;
  take_tables<T>(t, cp, cp + D / 2, sp, sp + D / 2);
  const auto row = [&](auto kind, int h, int heads) {
    constexpr int kKind = decltype(kind)::value;
    int64_t step;
    const T* p = row_source<T>(a, kKind, t.b, t.s, step) + t.c;
    p += h * step;
    const uint4 u1[1] = {*reinterpret_cast<const uint4*>(p)}, u2[1] = {*reinterpret_cast<const uint4*>(p + D / 2)};
    token_rows<T, CS, D, HALVES, kKind, 1>(a, t, h, 0, heads, u1, u2);
  };
  for (int r = threadIdx.x / kTpr; r < hq + 2 * hkv; r += kSlots) {
    if (r < hq)
      row(std::integral_constant<int, 0>(), r, hq);
    else if (r < hq + hkv)
      row(std::integral_constant<int, 1>(), r - hq, hkv);
    else
      row(std::integral_constant<int, 2>(), r - hq - hkv, hkv);
  }
}

template <typename T, typename CS, int D, bool HALVES>
__global__ void __launch_bounds__(32 * kPromptWarps, kPromptCtas)
    paged_append_int4_prompt_kernel(const __grid_constant__ aicas_paged_append_int4_params a) {
  using K = Token<CS, D>;
  constexpr int kTpr = K::kTpr, kSlots = 32 / kTpr, kRows = 2 * kSlots;  // rows of a unit
  __shared__ uint4 ring[kPromptWarps][kUnits][4][32];  // [first and second half of row 0, of row 1]
  constexpr int kTabVecs = K::kV * (int)sizeof(CS) / 16;
  __shared__ uint4 tables[kPromptWarps][32][4 * kTabVecs + 1];  // a lane's cos and sin; 1: to turn the banks
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, r0 = lane / kTpr;
  const int tokens = a.batch * a.seq_len, warps = (int)gridDim.x * kPromptWarps;
  const int hq = a.num_q_heads, hkv = a.num_kv_heads, nq = (hq + kRows - 1) / kRows, nk = (hkv + kRows - 1) / kRows;
  K t;
  t.c = lane % kTpr * K::kV;
  t.lanes = ((1u << kTpr) - 1u) << (r0 * kTpr);
  grid_launch_dependents();
  grid_dependency_wait();
  const int first = blockIdx.x * kPromptWarps + warp;
  // the unit that is copied next
  int64_t to_come = first;
  int unit = 0, b = 0, s = 0;
  const auto copy = [&](uint4 (&stage)[4][32]) {
    if (to_come < tokens) {
      if (unit == 0) b = (int)to_come / a.seq_len, s = (int)to_come - b * a.seq_len;
      const int kind = unit < nq ? 0 : unit < nq + nk ? 1 : 2, of_kind = unit - (kind == 0 ? 0 : kind == 1 ? nq : nq + nk);
      int64_t step;
      const T* src = row_source<T>(a, kind, b, s, step) + t.c;
      const int h = of_kind * kRows + r0, heads = kind == 0 ? hq : hkv;
#pragma unroll
      for (int j = 0; j < 2; ++j)
        if (h + j * kSlots < heads) {
          const T* p = src + (h + j * kSlots) * step;
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(&stage[2 * j][lane])), "l"(p) : "memory");
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(&stage[2 * j + 1][lane])), "l"(p + D / 2) : "memory");
        }
      if (++unit == nq + 2 * nk) unit = 0, to_come += warps;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  uint4* const mine = tables[warp][lane];
  const auto copy_tables = [&](int b, int s) {
    const CS* from[2] = {static_cast<const CS*>(a.cos) + b * a.cs_stride_b + s * a.cs_stride_s + t.c,
                         static_cast<const CS*>(a.sin) + b * a.cs_stride_b + s * a.cs_stride_s + t.c};
#pragma unroll
    for (int e = 0; e < 4 * kTabVecs; ++e)
      asm volatile("cp.async.ca.shared.global [%0], [%1], 16;" ::"r"(smem_u32(mine + e)),
                   "l"(from[e / (2 * kTabVecs)] + e / kTabVecs % 2 * (D / 2) + e % kTabVecs * (16 / (int)sizeof(CS))) : "memory");
  };
  if (first >= tokens) return;
  t.b = first / a.seq_len, t.s = first - t.b * a.seq_len;
  copy_tables(t.b, t.s);  // in the first unit's group
#pragma unroll
  for (int k = 0; k < kUnits; ++k) copy(ring[warp][k]);
  int2 place = place_of(a, t.b, t.s, lane == 0);
  int at = 0;
  const auto rows = [&](auto kind, int n, int heads) {
    constexpr int kKind = decltype(kind)::value;
#pragma unroll 1
    for (int u = 0; u < n; ++u) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kUnits - 1) : "memory");
      uint4(&stage)[4][32] = ring[warp][at];
      const uint4 u1[2] = {stage[0][lane], stage[2][lane]}, u2[2] = {stage[1][lane], stage[3][lane]};
      token_rows<T, CS, D, HALVES, kKind, 2>(a, t, u * kRows + r0, kSlots, heads, u1, u2);
      copy(stage);
      at = at + 1 == kUnits ? 0 : at + 1;
    }
  };
#pragma unroll 1
  for (int64_t token = first; token < tokens;) {
    // the tables' group is not the last one
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    const CS* tab = reinterpret_cast<const CS*>(mine);
    constexpr int kEach = K::kV;
    take_tables<T>(t, tab, tab + kEach, tab + 2 * kEach, tab + 3 * kEach);
    t.page = place.x, t.row = place.y;
    rows(std::integral_constant<int, 0>(), nq, hq);
    token += warps;
    const int nb = token < tokens ? (int)token / a.seq_len : t.b, ns = token < tokens ? (int)token - nb * a.seq_len : t.s;
    if (token < tokens) {
      copy_tables(nb, ns);  // q's rows are done, so these are read; they go into the next unit's group
      place = place_of(a, nb, ns, lane == 0);
    }
    rows(std::integral_constant<int, 1>(), nk, hkv);
    rows(std::integral_constant<int, 2>(), nk, hkv);
    t.b = nb, t.s = ns;
  }
}

// Tokens up to which each gets a CTA: the append and read of 16 x 16 tokens of 8 KV heads
// 5.3 us, a warp each 7.3; of 512 8.4, 11.1; of 1024 13.2, 12.7; of 2 x 2048 45.8, 24.3.
constexpr int kPromptTokens = 600;

template <typename T, typename CS, int D, bool HALVES>
cudaError_t launch_append_sized(const aicas_paged_append_int4_params& p, int sms, cudaStream_t st) {
  const int64_t tokens = (int64_t)p.batch * p.seq_len;
  if (tokens <= kPromptTokens)
    return launch_pdl(paged_append_int4_kernel<T, CS, D, HALVES>, dim3((unsigned)tokens), dim3(256), 0, st, p);
  const int64_t ctas = (tokens + kPromptWarps - 1) / kPromptWarps;
  return launch_pdl(paged_append_int4_prompt_kernel<T, CS, D, HALVES>, dim3((unsigned)(ctas < kPromptCtas * sms ? ctas : kPromptCtas * sms)),
                    dim3(32 * kPromptWarps), 0, st, p);
}

template <typename T, typename CS>
cudaError_t launch_append(const aicas_paged_append_int4_params& p, int sms, cudaStream_t st) {
  if (p.head_dim == 64) return launch_append_sized<T, CS, 64, false>(p, sms, st);
  return p.group_size == 64 ? launch_append_sized<T, CS, 128, true>(p, sms, st) : launch_append_sized<T, CS, 128, false>(p, sms, st);
}

// ------------------------------------------------------------------ reads

// 4 bytes of codes and the row's pair to 8 elements.
template <typename T>
__device__ __forceinline__ uint4 widened(uint32_t u, uint32_t p) {
  union {
    uint32_t u;
    T t[2];
  } pair;
  pair.u = p;
  const float scale = Elem<T>::to_float(pair.t[0]), least = Elem<T>::to_float(pair.t[1]);
  // a byte below the exponent of 2^23 is 2^23 and the byte
  constexpr float kWhole = 8388608.f;
  const Two by(scale), from(least);
  const uint32_t even = u & 0x0f0f0f0fu, odd = u >> 4 & 0x0f0f0f0fu;
  float f[8];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const Two code(__uint_as_float(__byte_perm(even, 0x4b000000u, 0x7440 + k)), __uint_as_float(__byte_perm(odd, 0x4b000000u, 0x7440 + k)));
    fma2(code + Two(-kWhole), by, from).get(f[2 * k], f[2 * k + 1]);
  }
  return pack_vec<T>(f);
}

// n / (page_size / 8) for n < 2^28, as in paged_int4_tiles.cuh.
struct ByOctets {
  uint32_t mul;
  int shift;
};
ByOctets by_octets(int page_size) {
  const int octets = page_size / 8;
  int shift = 0;
  while ((1ll << shift) < octets) ++shift;
  return {(uint32_t)((((1ull << shift) - octets) << 32) / octets + 1), shift};
}

// The row of slot pos + s, if it is to be read: page (else -1) and row in it.
__device__ __forceinline__ int2 row_at(const aicas_paged_read_int4_params& a, ByOctets by, int b, int pos, int fresh, int s) {
  const long long slot = (long long)pos + s;
  if (s >= fresh || slot < 0 || slot >= a.max_pages * a.page_size) return make_int2(-1, 0);
  const uint32_t n = (uint32_t)slot >> 3, i = (__umulhi(n, by.mul) + n) >> by.shift;
  const int page = a.page_table[b * a.table_stride + i];
  return make_int2(page < a.num_pages ? page : -1, (int)((uint32_t)slot - i * (uint32_t)a.page_size));
}

// HBM bound, by what it writes: 16 elements a thread, 8 bytes of codes in and 32 bytes out, of
// ROWS rows of one request, side and head, so that their page numbers, codes and pairs are on
// the way at once.
template <typename T, int D, bool HALVES, int ROWS>
__global__ void __launch_bounds__(256) paged_read_int4_kernel(const __grid_constant__ aicas_paged_read_int4_params a, ByOctets by, int chunks) {
  constexpr int kTpr = D / 16, kSlots = 256 / kTpr;
  const int b = blockIdx.x / chunks, h = blockIdx.y >> 1, side = blockIdx.y & 1;
  const int c = threadIdx.x % kTpr * 16, s0 = (blockIdx.x - b * chunks) * kSlots * ROWS + threadIdx.x / kTpr;
  grid_launch_dependents();
  grid_dependency_wait();
  const int fresh = a.num_tokens != nullptr ? min(a.num_tokens[b], a.seq_len) : a.seq_len;
  const int pos = a.positions[b];
  const aicas_int4_pages& from = a.kv[side];
  const uint8_t* codes = static_cast<const uint8_t*>(from.codes) + h * from.cs_h + c / 2;
  const T* pairs = static_cast<const T*>(from.scales) + h * from.ss_h + (HALVES && c >= D / 2 ? 2 : 0);
  int2 at[ROWS];
#pragma unroll
  for (int j = 0; j < ROWS; ++j) at[j] = row_at(a, by, b, pos, fresh, s0 + j * kSlots);
  uint2 u[ROWS];
  uint32_t p[ROWS];
#pragma unroll
  for (int j = 0; j < ROWS; ++j) {
    u[j] = make_uint2(0, 0), p[j] = 0;
    if (at[j].x >= 0) {
      u[j] = *reinterpret_cast<const uint2*>(codes + at[j].x * from.cs_p + at[j].y * from.cs_t);
      p[j] = *reinterpret_cast<const uint32_t*>(pairs + at[j].x * from.ss_p + at[j].y * from.ss_t);
    }
  }
  T* out = static_cast<T*>(a.out[side]) + b * a.out_stride_b + h * a.out_stride_h + c;
#pragma unroll
  for (int j = 0; j < ROWS; ++j) {
    const int s = s0 + j * kSlots;
    if (s >= a.seq_len) break;
    uint4* to = reinterpret_cast<uint4*>(out + (int64_t)s * a.out_stride_s);
    to[0] = widened<T>(u[j].x, p[j]);
    to[1] = widened<T>(u[j].y, p[j]);
  }
}

// The few rows of a decode step: all of a request's at once, in CTAs of kFewThreads.
constexpr int kFewThreads = 32;

template <typename T, int D, bool HALVES>
__global__ void __launch_bounds__(kFewThreads) paged_read_few_int4_kernel(const __grid_constant__ aicas_paged_read_int4_params a, ByOctets by) {
  constexpr int kTpr = D / 8;
  const int b = blockIdx.x, c = threadIdx.x % kTpr * 8;
  grid_launch_dependents();
  grid_dependency_wait();
  const int fresh = a.num_tokens != nullptr ? min(a.num_tokens[b], a.seq_len) : a.seq_len;
  const int pos = a.positions[b];
  const int r = (blockIdx.y * kFewThreads + threadIdx.x) / kTpr;
  if (r < 2 * a.num_kv_heads * a.seq_len) {
    const int head = a.seq_len == 1 ? r : r / a.seq_len, s = r - head * a.seq_len, h = head >> 1, side = head & 1;
    const aicas_int4_pages& from = a.kv[side];
    const int2 at = row_at(a, by, b, pos, fresh, s);
    uint32_t u = 0, p = 0;
    if (at.x >= 0) {
      u = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(from.codes) + at.x * from.cs_p + h * from.cs_h +
                                             at.y * from.cs_t + c / 2);
      p = *reinterpret_cast<const uint32_t*>(static_cast<const T*>(from.scales) + at.x * from.ss_p + h * from.ss_h +
                                             at.y * from.ss_t + (HALVES && c >= D / 2 ? 2 : 0));
    }
    *reinterpret_cast<uint4*>(static_cast<T*>(a.out[side]) + b * a.out_stride_b + h * a.out_stride_h + s * a.out_stride_s + c) =
        widened<T>(u, p);
  }
}

template <typename T, int D, bool HALVES>
cudaError_t launch_read_sized(const aicas_paged_read_int4_params& p, cudaStream_t st) {
  // with the append of as many: 16 x 16 tokens of 8 heads (2048) 5.3 us, 5.7 in the other kernel, 256 x 1 5.5, 8.5;
  // 1 x 512 (65536) 9.0, 8.1
  if ((int64_t)p.num_kv_heads * p.seq_len * (D / 8) <= 2048)
    return launch_pdl(paged_read_few_int4_kernel<T, D, HALVES>,
                      dim3((unsigned)p.batch, (2 * p.num_kv_heads * p.seq_len * (D / 8) + kFewThreads - 1) / kFewThreads), dim3(kFewThreads), 0,
                      st, p, by_octets(p.page_size));
  const int64_t rows = 256 / (D / 16) * 2, chunks = (p.seq_len + rows - 1) / rows;
  const dim3 grid((unsigned)(chunks * p.batch), 2u * p.num_kv_heads);
  return launch_pdl(paged_read_int4_kernel<T, D, HALVES, 2>, grid, dim3(256), 0, st, p, by_octets(p.page_size), (int)chunks);
}

template <typename T>
cudaError_t launch_read(const aicas_paged_read_int4_params& p, cudaStream_t st) {
  if (p.head_dim == 64) return launch_read_sized<T, 64, false>(p, st);
  return p.group_size == 64 ? launch_read_sized<T, 128, true>(p, st) : launch_read_sized<T, 128, false>(p, st);
}

int status(cudaError_t e, const char* what, char* err, size_t errlen) {
  if (e == cudaSuccess) return AICAS_OK;
  snprintf(err, errlen, "%s launch: %s (%s)", what, cudaGetErrorString(e), cudaGetErrorName(e));
  return AICAS_ERR_CUDA;
}

}  // namespace

int run_paged_append_int4(const aicas_paged_append_int4_params* p, int sms, cudaStream_t stream, char* err, size_t errlen) {
  const bool f32cs = p->cs_dtype == AICAS_DTYPE_F32;
  cudaError_t e = cudaErrorInvalidValue;
  if (p->dtype == AICAS_DTYPE_F16)
    e = f32cs ? launch_append<__half, float>(*p, sms, stream) : launch_append<__half, __half>(*p, sms, stream);
  else if (p->dtype == AICAS_DTYPE_BF16)
    e = f32cs ? launch_append<__nv_bfloat16, float>(*p, sms, stream) : launch_append<__nv_bfloat16, __nv_bfloat16>(*p, sms, stream);
  return status(e, "paged 4-bit append", err, errlen);
}

int run_paged_read_int4(const aicas_paged_read_int4_params* p, cudaStream_t stream, char* err, size_t errlen) {
  return status(p->dtype == AICAS_DTYPE_F16 ? launch_read<__half>(*p, stream) : launch_read<__nv_bfloat16>(*p, stream),
                "paged 4-bit read", err, errlen);
}

}  // namespace aicas
