// 8-bit operands for the block-scaled product (sm_100a): quantizers of
// activation rows and of weights, the gated activation and the RMS norm with
// the residual's addition, each writing e4m3 values and fp32 scales.
//
// For a block B of values y (1 x 128 columns, or 128 x 128 for weights):
//   amax = max(2^-100, max |y|)      scale = amax / 448      q = e4m3(448 y / amax)
// 448 is the largest e4m3 value, so nothing saturates; the quotient is formed in
// fp32 (by the quantizers with a residual step, by norm and gate, whose y carry
// roundings already, as one product with 448 / amax) and rounded to even.  NaN in
// a block makes amax, hence the whole block, NaN; an infinity makes scale
// infinite, its own value NaN and the others 0.  The floor 2^-100 keeps the
// reciprocal finite: blocks below it (zeros above all) give q = 0 or values
// that small a scale can hold.
//
// All of them read each input once and write each output once, so the bound
// is HBM; sums and statistics are fp32.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "fp8_launch.cuh"
#include "llvq_b200.h"
#include "llvq_internal.h"

namespace llvq {

namespace {

constexpr int kVec = 16;                         // elements a thread handles at a time
constexpr int kGroup = kFp8Block / kVec;         // 8 threads share one block of 128 columns
constexpr float kE4m3Max = 448.f;
constexpr float kAmaxFloor = 0x1p-100f;

// Two fp32 values in a register pair: one instruction works on both.  The
// kernels are as near to the issue rate as to the memory's (swiglu of 4096 x
// 11008 issued in 81% of the cycles), so what they compute is written in pairs.
struct F2 {
  uint64_t v;
};

__device__ __forceinline__ F2 pair(float lo, float hi) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ F2 pair(float both) { return pair(both, both); }
__device__ __forceinline__ float2 halves(F2 a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
  return r;
}
__device__ __forceinline__ F2 fma(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ F2 operator*(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 operator+(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}

constexpr int kPairs = kVec / 2;

// Sixteen elements as they lie in memory: pairs of 16-bit values, or fp32.
template <typename T>
struct Raw {
  static constexpr int kWords = kVec * (int)sizeof(T) / 4;
  uint32_t w[kWords];
};

// The two 16-bit values of a word.
template <typename T>
__device__ __forceinline__ F2 pair_in(uint32_t word) {
  static_assert(sizeof(T) == 2);
  if constexpr (std::is_same_v<T, __half>) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&word));
    return pair(f.x, f.y);
  } else {
    return pair(__uint_as_float(word << 16), __uint_as_float(word & 0xFFFF0000u));
  }
}

template <typename T>
__device__ __forceinline__ void unpack(const Raw<T>& r, F2 (&v)[kPairs]) {
#pragma unroll
  for (int i = 0; i < kPairs; ++i) {
    if constexpr (sizeof(T) == 4) v[i] = pair(__uint_as_float(r.w[2 * i]), __uint_as_float(r.w[2 * i + 1]));
    else v[i] = pair_in<T>(r.w[i]);
  }
}

template <typename T>
__device__ __forceinline__ Raw<T> pack(const F2 (&v)[kPairs]) {
  Raw<T> r;
#pragma unroll
  for (int i = 0; i < kPairs; ++i) {
    const float2 f = halves(v[i]);
    if constexpr (sizeof(T) == 4) {
      r.w[2 * i] = __float_as_uint(f.x);
      r.w[2 * i + 1] = __float_as_uint(f.y);
    } else if constexpr (std::is_same_v<T, __half>) {
      const __half2 h = __floats2half2_rn(f.x, f.y);
      r.w[i] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
      r.w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  return r;
}

// Sixteen elements, those from `valid` on as zeros.  kStep elements are loaded
// at a time (8 or 4: every step starts on its boundary, 16 bytes at most, and
// the columns are a multiple of it), by predicated loads without branches, so
// that all the loads of a thread are in flight together.
// Plain loads, no __restrict__ on the pointers they come from and no read-only
// path: this kernel starts while the one ahead of it may still write what p points
// to, so nothing is constant for the kernel's lifetime and no load may be moved
// ahead of wait_for_inputs().
template <typename T, int kStep>
__device__ __forceinline__ Raw<T> load_vec(const T* p, int valid) {
  Raw<T> r;
  if constexpr (kStep * sizeof(T) >= 16) {
#pragma unroll
    for (int i = 0; i < Raw<T>::kWords / 4; ++i) {
      const uint4 q = i * 16 < valid * (int)sizeof(T) ? reinterpret_cast<const uint4*>(p)[i] : make_uint4(0, 0, 0, 0);
      r.w[4 * i] = q.x, r.w[4 * i + 1] = q.y, r.w[4 * i + 2] = q.z, r.w[4 * i + 3] = q.w;
    }
  } else if constexpr (kStep * sizeof(T) == 8) {
#pragma unroll
    for (int i = 0; i < Raw<T>::kWords / 2; ++i) {
      const uint2 q = i * 8 < valid * (int)sizeof(T) ? reinterpret_cast<const uint2*>(p)[i] : make_uint2(0, 0);
      r.w[2 * i] = q.x, r.w[2 * i + 1] = q.y;
    }
  }
  return r;
}

template <typename T, int kStep>
__device__ __forceinline__ void store_vec(T* p, const Raw<T>& r, int valid) {
  if constexpr (kStep * sizeof(T) >= 16) {
#pragma unroll
    for (int i = 0; i < Raw<T>::kWords / 4; ++i)
      if (i * 16 < valid * (int)sizeof(T))
        reinterpret_cast<uint4*>(p)[i] = make_uint4(r.w[4 * i], r.w[4 * i + 1], r.w[4 * i + 2], r.w[4 * i + 3]);
  } else if constexpr (kStep * sizeof(T) == 8) {
#pragma unroll
    for (int i = 0; i < Raw<T>::kWords / 2; ++i)
      if (i * 8 < valid * (int)sizeof(T)) reinterpret_cast<uint2*>(p)[i] = make_uint2(r.w[2 * i], r.w[2 * i + 1]);
  }
}

// Where nothing is known of the boundaries (kStep 1): a warp's four blocks of 128
// columns in loads and stores of one element a lane, neighbours side by side, turned
// through 1 KB of the warp's shared memory into sixteen elements a thread and back.
// (Loads of a thread's own columns touched 32 sectors each: 8000 x 4097 bf16 norm
// with a residual 216 us against 84, rows 47 against 24, gate 79 against 42,
// 128 x 128 blocks 38 against 27.)
// unit(u, &left): block u's first element and its columns in the matrix, 0..128.
constexpr int kTurnBytes = 1024;

template <typename T>
using Bits = std::conditional_t<sizeof(T) == 4, uint32_t, uint16_t>;

// The loads, all in flight together ...
template <typename T>
struct Loaded {
  Bits<T> v[kVec];
  template <typename Unit>
  __device__ __forceinline__ explicit Loaded(Unit unit) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      int left;
      const Bits<T>* p = reinterpret_cast<const Bits<T>*>(unit(u, left));
#pragma unroll
      for (int j = 0; j < 4; ++j) v[u * 4 + j] = j * 32 + lane < left ? p[j * 32 + lane] : (Bits<T>)0;
    }
  }
};

// ... and what they brought, as the threads work on it.
template <typename T>
__device__ __forceinline__ Raw<T> turned(uint8_t* turn, const Loaded<T>& in) {
  constexpr int kUnits = kTurnBytes / (kFp8Block * (int)sizeof(T));  // blocks a pass, of 4
  const int lane = threadIdx.x & 31;
  Raw<T> r;
#pragma unroll
  for (int pass = 0; pass < 4 / kUnits; ++pass) {
    __syncwarp();  // what was there before has been read
#pragma unroll
    for (int i = 0; i < kUnits * 4; ++i) reinterpret_cast<Bits<T>*>(turn)[i * 32 + lane] = in.v[pass * kUnits * 4 + i];
    __syncwarp();
    if (lane / (kUnits * kGroup) == pass) {
#pragma unroll
      for (int i = 0; i < Raw<T>::kWords / 4; ++i) {
        const uint4 q = reinterpret_cast<const uint4*>(turn)[(lane % (kUnits * kGroup)) * (Raw<T>::kWords / 4) + i];
        r.w[4 * i] = q.x, r.w[4 * i + 1] = q.y, r.w[4 * i + 2] = q.z, r.w[4 * i + 3] = q.w;
      }
    }
  }
  return r;
}

template <typename T, typename Unit>
__device__ __forceinline__ void store_turned(uint8_t* turn, const Raw<T>& r, Unit unit) {
  constexpr int kUnits = kTurnBytes / (kFp8Block * (int)sizeof(T));
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int pass = 0; pass < 4 / kUnits; ++pass) {
    __syncwarp();
    if (lane / (kUnits * kGroup) == pass) {
#pragma unroll
      for (int i = 0; i < Raw<T>::kWords / 4; ++i)
        reinterpret_cast<uint4*>(turn)[(lane % (kUnits * kGroup)) * (Raw<T>::kWords / 4) + i] =
            make_uint4(r.w[4 * i], r.w[4 * i + 1], r.w[4 * i + 2], r.w[4 * i + 3]);
    }
    __syncwarp();
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      int left;
      Bits<T>* p = reinterpret_cast<Bits<T>*>(unit(pass * kUnits + u, left));
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j * 32 + lane < left) p[j * 32 + lane] = reinterpret_cast<const Bits<T>*>(turn)[(u * 4 + j) * 32 + lane];
    }
  }
}

__device__ __forceinline__ float2 both(__half2 v) { return __half22float2(v); }
__device__ __forceinline__ float2 both(__nv_bfloat162 v) { return __bfloat1622float2(v); }

// max |.| that keeps NaN (fmaxf would drop it).
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ float amax_of(const F2 (&v)[kPairs]) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < kPairs; ++i) {
    const float2 f = halves(v[i]);
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(m), "f"(f.x), "f"(f.y));
  }
  return m;
}

// The same of the values as they lie in memory: pairs at a time (their largest
// magnitude is one of them, so nothing is rounded).
template <typename T>
__device__ __forceinline__ float amax_of(const Raw<T>& r) {
  if constexpr (sizeof(T) == 4) {
    F2 v[kPairs];
    unpack(r, v);
    return amax_of(v);
  } else {
    using T2 = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
    T2 m = __habs2(*reinterpret_cast<const T2*>(&r.w[0]));
#pragma unroll
    for (int i = 1; i < Raw<T>::kWords; ++i) m = __hmax2_nan(m, __habs2(*reinterpret_cast<const T2*>(&r.w[i])));
    const float2 f = both(m);
    return max_nan(f.x, f.y);
  }
}

// Largest of the 8 threads that share a block.
__device__ __forceinline__ float group_max(float m) {
#pragma unroll
  for (int o = kGroup / 2; o; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  return m;
}

__device__ __forceinline__ float floored(float amax) { return max_nan(amax, kAmaxFloor); }

// RN(amax / 448): one residual step from the rounded reciprocal (Markstein 1990).
__device__ __forceinline__ float scale_of(float amax) {
  constexpr float kInv = 1.f / kE4m3Max;
  const float q = amax * kInv;
  return isinf(q) ? q : fmaf(fmaf(-q, kE4m3Max, amax), kInv, q);
}

// 1 / d within one unit: the approximate reciprocal and a Newton step (d normal, not near the ends of the range).
__device__ __forceinline__ float reciprocal(float d) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
  return fmaf(r, fmaf(-d, r, 1.f), r);
}

// 1 / sqrt(v) within two units, from the approximate root and a Newton step;
// infinite for 0, 0 for infinity.
__device__ __forceinline__ float inverse_root(float v) {
  float r;
  asm("rsqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(v));
  const float better = fmaf(fmaf(-v * r, r, 1.f), 0.5f * r, r);
  return v > 0x1p-126f && v < 0x1p126f ? better : r;
}

// 448 v / amax for values v that fp32 holds exactly: q0 = z r with z = 448 v
// (exact for 16-bit inputs; fp32 ones carry a rounding of 2^-24 from here on) and
// r = 1 / amax, and one residual step, q = q0 + (z - q0 amax) r (Markstein 1990).
//  Inputs of few bits lie on ties of e4m3
// often, and there the residual is exact and q is the tie itself, so that it
// is rounded to even as it should; a quotient off by one unit would fall on
// either side.  448 and amax are both taken times 2^-64 where 448 amax could
// overflow; an infinite amax gives 0 for finite values and NaN for infinite ones.
struct ExactQuotient {
  F2 mul, r, minus_d;
  float scale;
  __device__ __forceinline__ explicit ExactQuotient(float amax) {
    amax = floored(amax);
    scale = scale_of(amax);
    const bool big = amax > 0x1p100f;
    const float d = big ? amax * 0x1p-64f : amax;
    const bool infinite = isinf(amax);
    mul = pair(big ? kE4m3Max * 0x1p-64f : kE4m3Max);
    r = pair(infinite ? 0.f : reciprocal(d));
    minus_d = pair(infinite ? 0.f : -d);
  }
  __device__ __forceinline__ F2 operator()(F2 v) const {
    const F2 z = v * mul, q = z * r;
    return fma(fma(q, minus_d, z), r, q);
  }
};

// 448 v / amax for values that carry fp32 roundings themselves: one product
// with 448 / amax.
struct Quotient {
  F2 r;
  float scale;
  __device__ __forceinline__ explicit Quotient(float amax) {
    amax = floored(amax);
    scale = scale_of(amax);
    const bool big = amax > 0x1p100f;
    const float q = reciprocal(big ? amax * 0x1p-64f : amax) * (big ? kE4m3Max * 0x1p-64f : kE4m3Max);
    r = pair(isinf(amax) ? 0.f : q);
  }
  __device__ __forceinline__ F2 operator()(F2 v) const { return v * r; }
};

// Two e4m3 bytes, lo in the low one.
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// Sixteen values as e4m3; rows start on 16-byte boundaries.
template <typename Q>
__device__ __forceinline__ void store_q(uint8_t* p, const F2 (&v)[kPairs], const Q& quo, int valid) {
  uint32_t w[kVec / 4];
#pragma unroll
  for (int i = 0; i < kVec / 4; ++i) {
    const float2 lo = halves(quo(v[2 * i])), hi = halves(quo(v[2 * i + 1]));
    w[i] = e4m3x2(lo.x, lo.y) | e4m3x2(hi.x, hi.y) << 16;
  }
  if (valid >= kVec) {
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int i = 0; i < kVec; ++i)
      if (i < valid) p[i] = (uint8_t)(w[i >> 2] >> (8 * (i & 3)));
  }
}

__device__ __forceinline__ int valid_of(int64_t cols, int64_t c) {
  const int64_t left = cols - c;
  return left >= kVec ? kVec : left > 0 ? (int)left : 0;
}

// exp(-c) of a pair, c within +-88.5: 2^-n (1 + l ln 2), n = RN(c kLog2e) and l
// what that product and the rounded constant lost (kLog2e = log2 e - 1.926e-8,
// kTail = -1.926e-8 ln 2), so that its error is that of ex2.approx (2^-22) for
// every c; below 2^-126 it is 0.
__device__ __forceinline__ F2 exp_minus(F2 c) {
  constexpr float kLog2e = 1.44269504f, kLn2 = 0.693147181f, kTail = -1.33497582e-8f;
  const F2 n = c * pair(kLog2e);
  const F2 l = fma(c, pair(-kLog2e), n);
  const float2 m = halves(n);
  float2 e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(-m.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(-m.y));
  const F2 ee = pair(e.x, e.y);
  return fma(ee, fma(c, pair(kTail), l * pair(kLn2)), ee);
}

__device__ __forceinline__ F2 clamped(F2 v) {
  const float2 f = halves(v);
  return pair(fminf(fmaxf(f.x, -88.5f), 88.5f), fminf(fmaxf(f.y, -88.5f), 88.5f));
}

// gate / (1 + exp(-gate)) of a pair; the reciprocal takes one Newton step.  The
// exponent's argument is clamped so that all of this stays finite: below g =
// -87.3 the reciprocal is flushed to zero and the quotient g * 0 (NaN for an
// infinite g; low_gate() is for the finite ones), above 88.5 it is g.
__device__ __forceinline__ F2 silu(F2 g) {
  const F2 minus_d = fma(exp_minus(clamped(g)), pair(-1.f), pair(-1.f));
  const float2 d = halves(minus_d);
  float2 r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(-d.x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(-d.y));
  F2 rr = pair(r.x, r.y);
  rr = fma(rr, fma(minus_d, rr, pair(1.f)), rr);
  return g * rr;
}

// silu(gate) up for gates below kLowGate: exp(-gate) or its reciprocal leaves
// fp32's normal range there, and the product need not.  1 + exp(-gate) is
// exp(-gate) to the last bit, so with E = exp(gate / 2) it is (gate E) (E up).  E
// is 0 below gate = -174.7, where the product is below 2^-116 whatever up is.  A
// group of sixteen asks for its smallest gate first: 64 x 14336 bf16 3.2 us, 3.1
// without.
constexpr float kLowGate = -87.f;
__device__ __forceinline__ F2 low_gate(F2 gate, F2 up) {
  const F2 e = exp_minus(clamped(gate * pair(-0.5f)));
  return gate * e * (e * up);
}

// Smallest of the values as they lie in memory; NaN does not count.
template <typename T>
__device__ __forceinline__ float lowest_of(const Raw<T>& r) {
  if constexpr (sizeof(T) == 4) {
    float m = __uint_as_float(r.w[0]);
#pragma unroll
    for (int i = 1; i < Raw<T>::kWords; ++i) m = fminf(m, __uint_as_float(r.w[i]));
    return m;
  } else {
    using T2 = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
    T2 m = *reinterpret_cast<const T2*>(&r.w[0]);
#pragma unroll
    for (int i = 1; i < Raw<T>::kWords; ++i) m = __hmin2(m, *reinterpret_cast<const T2*>(&r.w[i]));
    const float2 f = both(m);
    return fminf(f.x, f.y);
  }
}

__device__ __forceinline__ F2 any_gate(F2 gate, F2 up) {
  const float2 g = halves(gate), low = halves(low_gate(gate, up)), y = halves(silu(gate) * up);
  return pair(g.x < kLowGate ? low.x : y.x, g.y < kLowGate ? low.y : y.y);
}

// any_gate of sixteen: a rolled loop that works on the first pair and moves the
// others up, results behind them, so that it takes no registers beside the inputs'.
template <typename T>
__device__ __forceinline__ void any_gates(F2 (&y)[kPairs], const Raw<T>& gate, const Raw<T>& up) {
  if constexpr (sizeof(T) == 2) {
    uint32_t a[kPairs], b[kPairs];
#pragma unroll
    for (int i = 0; i < kPairs; ++i) a[i] = gate.w[i], b[i] = up.w[i];
#pragma unroll 1
    for (int turn = 0; turn < kPairs; ++turn) {
      const float2 v = halves(any_gate(pair_in<T>(a[0]), pair_in<T>(b[0])));
#pragma unroll
      for (int i = 0; i + 1 < kPairs; ++i) a[i] = a[i + 1], b[i] = b[i + 1];
      a[kPairs - 1] = __float_as_uint(v.x), b[kPairs - 1] = __float_as_uint(v.y);
    }
#pragma unroll
    for (int i = 0; i < kPairs; ++i) y[i] = pair(__uint_as_float(a[i]), __uint_as_float(b[i]));
  } else {
    F2 w[kPairs];
    unpack(gate, y);
    unpack(up, w);
#pragma unroll 1
    for (int turn = 0; turn < kPairs; ++turn) {
      const F2 v = any_gate(y[0], w[0]);
#pragma unroll
      for (int i = 0; i + 1 < kPairs; ++i) y[i] = y[i + 1], w[i] = w[i + 1];
      y[kPairs - 1] = v;
    }
  }
}

// ---------------------------------------------------------------- rows
// Eight threads per (row, block of 128 columns), the next eight on the next
// block, so that every line is read and written whole; a thread loads all its
// kUnits units before it works on the first.  Sixteen elements a thread, not
// eight: what a thread spends once on a unit (three shuffles, the quotient, the
// addresses) was half of its instructions.  kGated: y = gate / (1 + exp(-gate)) * up.
constexpr int kRowThreads = 256;
template <typename T, bool kGated, int kStep>
constexpr int kRowUnits = sizeof(T) == 4 || kStep == 1 ? 1 : 2;

// CTAs an SM holds at least (0: not asked for).  4096 x 11008 gate, bf16: 37.6 us
// for four, 38.4 not asked for, 40.1 for five, which spill; fp32 59.1 for five, 75.9 for six.
template <typename T, bool kGated, int kStep>
constexpr int kRowCtas = !kGated || kStep == 1 ? 0 : sizeof(T) == 4 ? 5 : 4;

template <typename T, bool kGated, int kStep>
__global__ void __launch_bounds__(kRowThreads, kRowCtas<T, kGated, kStep>)
    rows_kernel(const T* x, int64_t ldx, const T* up, int64_t ldu, uint32_t rows, uint32_t blocks, uint32_t skip_rows,
                uint32_t skip_blocks, int64_t cols, Fp8Out out) {
  dependents_may_start();
  constexpr int kUnits = kRowUnits<T, kGated, kStep>;
  constexpr int kTeams = kRowThreads / kGroup;
  const uint32_t first = blockIdx.x * (kTeams * kUnits) + threadIdx.x / kGroup;
  const int in_block = (int)(threadIdx.x % kGroup) * kVec;
  uint32_t row[kUnits], b[kUnits];
  int valid[kUnits];
  Raw<T> rx[kUnits], ru[kUnits];
  wait_for_inputs();
#pragma unroll
  for (int j = 0; j < kUnits; ++j) {
    if (j == 0) {
      row[0] = first / blocks;
      b[0] = first - row[0] * blocks;
    } else {  // kTeams units on: skip_rows rows and skip_blocks blocks, without another division
      const uint32_t next = b[j - 1] + skip_blocks, wrap = next >= blocks;
      row[j] = row[j - 1] + skip_rows + wrap;
      b[j] = wrap ? next - blocks : next;
    }
    const int64_t c = (int64_t)b[j] * kFp8Block + in_block;
    valid[j] = row[j] < rows ? valid_of(cols, c) : 0;  // no early return: the whole warp meets in the shuffles
    if constexpr (kStep > 1) {
      rx[j] = load_vec<T, kStep>(x + (valid[j] ? row[j] * ldx + c : 0), valid[j]);
      if constexpr (kGated) ru[j] = load_vec<T, kStep>(up + (valid[j] ? row[j] * ldu + c : 0), valid[j]);
    } else {
      __shared__ alignas(16) uint8_t turn[kRowThreads / 32][kTurnBytes];
      const int64_t left = row[j] < rows ? cols - (int64_t)b[j] * kFp8Block : 0;
      auto load = [&](const T* m, int64_t ld) {
        const T* mine = m + (left > 0 ? row[j] * ld + (int64_t)b[j] * kFp8Block : 0);
        return Loaded<T>([&](int u, int& n) {
          n = __shfl_sync(0xffffffffu, (int)(left < kFp8Block ? left : kFp8Block), u * kGroup);
          return reinterpret_cast<const T*>(__shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(mine), u * kGroup));
        });
      };
      uint8_t* turning = turn[threadIdx.x / 32];
      const Loaded<T> lx = load(x, ldx);
      if constexpr (kGated) {
        const Loaded<T> lu = load(up, ldu);
        rx[j] = turned<T>(turning, lx);
        ru[j] = turned<T>(turning, lu);
      } else {
        rx[j] = turned<T>(turning, lx);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < kUnits; ++j) {
    F2 v[kPairs];
    float largest;
    if constexpr (kGated) {
      if (lowest_of(rx[j]) < kLowGate) {  // hardly ever
        any_gates(v, rx[j], ru[j]);
      } else {
        F2 w[kPairs];
        unpack(rx[j], v);
        unpack(ru[j], w);
#pragma unroll
        for (int i = 0; i < kPairs; ++i) v[i] = silu(v[i]) * w[i];
      }
      largest = amax_of(v);
    } else {
      unpack(rx[j], v);
      largest = amax_of(rx[j]);
    }
    const std::conditional_t<kGated, Quotient, ExactQuotient> quo(group_max(largest));
    if (!valid[j]) continue;
    store_q(out.q + row[j] * out.ld + (int64_t)b[j] * kFp8Block + in_block, v, quo, valid[j]);
    if (in_block == 0) out.scale[row[j] * out.scale_row + b[j] * out.scale_col] = quo.scale;
  }
}

// ---------------------------------------------------------------- 128 x 128 blocks
// One CTA per block: 256 threads hold its 16,384 values in registers (64 per
// thread, as they lie in memory) between the maximum and the store.
constexpr int kBlockThreads = 256;
constexpr int kBlockRowsPass = kBlockThreads / kGroup;       // 32 rows a pass
constexpr int kBlockPasses = kFp8Block / kBlockRowsPass;     // 4

template <typename T, int kStep>
__global__ void __launch_bounds__(kBlockThreads) blocks_kernel(const T* x, int64_t ldx, int64_t rows,
                                                               int64_t cols, uint32_t col_blocks, Fp8Out out) {
  dependents_may_start();
  __shared__ float red[kBlockThreads / 32];
  const uint32_t rb = blockIdx.x / col_blocks, cb = blockIdx.x % col_blocks;
  const int64_t c = (int64_t)cb * kFp8Block + (threadIdx.x % kGroup) * kVec;
  const int64_t r0 = (int64_t)rb * kFp8Block + threadIdx.x / kGroup;
  const int valid = valid_of(cols, c);
  Raw<T> raw[kBlockPasses];
  wait_for_inputs();
#pragma unroll
  for (int p = 0; p < kBlockPasses; ++p) {
    const int64_t r = r0 + p * kBlockRowsPass;
    if constexpr (kStep > 1) {
      const int live = r < rows ? valid : 0;
      raw[p] = load_vec<T, kStep>(x + (live ? r * ldx + c : 0), live);
    } else {
      __shared__ alignas(16) uint8_t turn[kBlockThreads / 32][kTurnBytes];
      const int64_t c0 = (int64_t)cb * kFp8Block, first = r - (threadIdx.x % 32) / kGroup;  // the warp's four rows
      const int width = (int)min(cols - c0, (int64_t)kFp8Block);
      const Loaded<T> in([&](int u, int& n) {
        n = first + u < rows ? width : 0;
        return x + (n ? (first + u) * ldx + c0 : 0);
      });
      raw[p] = turned<T>(turn[threadIdx.x / 32], in);
    }
  }
  float m = 0.f;
#pragma unroll
  for (int p = 0; p < kBlockPasses; ++p) m = max_nan(m, amax_of(raw[p]));
#pragma unroll
  for (int o = 16; o; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kBlockThreads / 32; ++w) m = max_nan(m, red[w]);
  const ExactQuotient quo(m);
#pragma unroll
  for (int p = 0; p < kBlockPasses; ++p) {
    const int64_t r = r0 + p * kBlockRowsPass;
    if (r < rows && valid) {
      F2 v[kPairs];
      unpack(raw[p], v);
      store_q(out.q + r * out.ld + c, v, quo, valid);
    }
  }
  if (threadIdx.x == 0) out.scale[rb * out.scale_row + cb * out.scale_col] = quo.scale;
}

// ---------------------------------------------------------------- RMS norm
// A CTA takes rows blockIdx.x, + gridDim.x, ...; a row stays in registers
// (kChunks groups of sixteen per thread) between the sum of squares and the 8-bit
// store, and the next row's loads are under way meanwhile:
//   h = x + residual (fp32; hidden = h rounded once)    y = h rsqrt(mean h^2 + eps) weight
// The norm uses the unrounded sum h.  Threads past the row hold zeros.
// Three shapes: up to 8192 columns one chunk, up to 16,384 two, with at most 512
// threads and the next row in registers; beyond, two chunks of up to 1024
// threads, which leave no registers for it.  (Rows on odd boundaries: norm_typed.)  (One chunk of 688 threads, for 11008
// columns, left an SM with a single CTA: 63 us against the two chunks' 58 for
// 4096 rows.)  8192 x 4096 with a residual runs at 6.3 TB/s.
// Registers a thread.  Nothing is spilled (8 bytes for fp32 above 16,384 columns
// with a residual) where vectors are loaded; rows on odd boundaries spill up to 408 bytes at
// 16,384 columns at most and 256 to 1416 beyond, where 1024 threads leave 64 registers each.
constexpr int norm_regs(int chunks, int threads, int step) {
  return threads == 1024 ? 64 : chunks == 2 ? 88 : step == 1 ? 80 : 64;
}

template <typename T, typename W, int kChunks, int kThreads, bool kResidual, int kStep>
__global__ void __maxnreg__(norm_regs(kChunks, kThreads, kStep))
    rms_norm_kernel(const T* x, int64_t ldx, const T* residual, int64_t ldr, const W* weight, float eps,
                    float inv_cols, int64_t rows, int64_t cols, T* hidden, int64_t ldh, Fp8Out out) {
  constexpr bool kAhead = kThreads == 512 && sizeof(T) == 2 && kStep > 1;  // fp32 rows would spill
  // The next row's loads go out ahead of the barrier, or behind it where a
  // residual's would spill (8192 x 4096: 37.2 us against 39.3; without a residual
  // 20.0 against 18.9).
  constexpr bool kLate = kChunks == 1 && kResidual;
  dependents_may_start();
  __shared__ float red[2][32];
  extern __shared__ __align__(16) uint8_t turn[];  // kTurnBytes a warp (kStep 1)
  // the four blocks of this warp in chunk j of a row that starts at p
  auto blocks_of = [&](auto* p, int j) {
    const int64_t c0 = (((int64_t)j * blockDim.x + threadIdx.x) & ~31LL) * kVec;
    return [p, c0, cols](int u, int& n) {
      const int64_t c = c0 + u * kFp8Block, left = cols - c;
      n = left <= 0 ? 0 : left < kFp8Block ? (int)left : kFp8Block;
      return p + (n ? c : 0);
    };
  };
  uint8_t* mine = turn + threadIdx.x / 32 * kTurnBytes;
  Raw<T> rx[kChunks], rr[kChunks];
  auto load = [&](int64_t row) {
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
      const int64_t c = ((int64_t)j * blockDim.x + threadIdx.x) * kVec;
      const int valid = row < rows ? valid_of(cols, c) : 0;
      if constexpr (kStep > 1) {
        rx[j] = load_vec<T, kStep>(x + (valid ? row * ldx + c : 0), valid);
        if constexpr (kResidual) rr[j] = load_vec<T, kStep>(residual + (valid ? row * ldr + c : 0), valid);
      }
    }
  };
  wait_for_inputs();
  if constexpr (kAhead) load(blockIdx.x);
  // the weights of a single chunk stay in registers where those reach
  constexpr bool kHold = kChunks == 1 && !(kAhead && kResidual);
  Raw<W> rw;
  auto load_weight = [&](int j) {
    const int64_t c = ((int64_t)j * blockDim.x + threadIdx.x) * kVec;
    const int valid = valid_of(cols, c);
    if constexpr (kStep > 1) rw = load_vec<W, kStep>(weight + (valid ? c : 0), valid);
    else rw = turned<W>(mine, Loaded<W>(blocks_of(weight, j)));
  };
  if constexpr (kHold) load_weight(0);
  int side = 0;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x, side ^= 1) {
    F2 h[kChunks][kPairs], squares = pair(0.f);
    if constexpr (!kAhead && kStep > 1) load(row);
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
      if constexpr (kStep == 1) {
        // one after the other: both in flight would spill (2047 x 16001 with a residual 107 us against 87)
        rx[j] = turned<T>(mine, Loaded<T>(blocks_of(x + row * ldx, j)));
        if constexpr (kResidual) rr[j] = turned<T>(mine, Loaded<T>(blocks_of(residual + row * ldr, j)));
      }
      unpack(rx[j], h[j]);
      if constexpr (kResidual) {
        F2 r[kPairs];
        unpack(rr[j], r);
#pragma unroll
        for (int i = 0; i < kPairs; ++i) h[j][i] = h[j][i] + r[i];
      }
#pragma unroll
      for (int i = 0; i < kPairs; ++i) squares = fma(h[j][i], h[j][i], squares);
    }
    float ss = halves(squares).x + halves(squares).y;
    if constexpr (kResidual) {
#pragma unroll
      for (int j = 0; j < kChunks; ++j) {
        const int64_t c = ((int64_t)j * blockDim.x + threadIdx.x) * kVec;
        const int valid = valid_of(cols, c);
        if constexpr (kStep > 1) store_vec<T, kStep>(hidden + (valid ? row * ldh + c : 0), pack<T>(h[j]), valid);
        else store_turned<T>(mine, pack<T>(h[j]), blocks_of(hidden + row * ldh, j));
      }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if ((threadIdx.x & 31) == 0) red[side][threadIdx.x >> 5] = ss;
    if constexpr (kAhead && !kLate) load(row + gridDim.x);
    __syncthreads();  // the other side is written next: one barrier a row
    // every warp adds the warps' sums in the same tree
    float total = (threadIdx.x & 31) < blockDim.x / 32 ? red[side][threadIdx.x & 31] : 0.f;
#pragma unroll
    for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    if constexpr (kAhead && kLate) load(row + gridDim.x);
    const float var = fmaf(total, inv_cols, eps);
    const float rstd = inverse_root(var);
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
      const int64_t c = ((int64_t)j * blockDim.x + threadIdx.x) * kVec;
      const int valid = valid_of(cols, c);
      if constexpr (!kHold) load_weight(j);
      F2 y[kPairs];
      unpack(rw, y);
#pragma unroll
      for (int i = 0; i < kPairs; ++i) y[i] = h[j][i] * pair(rstd) * y[i];
      const Quotient quo(group_max(amax_of(y)));
      if (valid) store_q(out.q + row * out.ld + c, y, quo, valid);
      if (valid && threadIdx.x % kGroup == 0)
        out.scale[row * out.scale_row + c / kFp8Block * out.scale_col] = quo.scale;
    }
  }
}

// The elements of a matrix that can be loaded at a time: 8, 4 or 1 (load_vec).
template <typename T>
int step_of(const void* p, int64_t ld, int64_t cols) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(p) | (uintptr_t)(ld * (int64_t)sizeof(T));
  const uintptr_t wide = sizeof(T) * 8 > 16 ? 16 : sizeof(T) * 8, half = sizeof(T) * 4;
  return at % wide == 0 && cols % 8 == 0 ? 8 : at % half == 0 && cols % 4 == 0 ? 4 : 1;
}

template <typename T, bool kGated, int kStep>
cudaError_t rows_step(Fp8In x, Fp8In up, int64_t rows, int64_t cols, Fp8Out out, cudaStream_t stream) {
  const int64_t blocks = (cols + kFp8Block - 1) / kFp8Block, units = rows * blocks;
  constexpr int kTeams = kRowThreads / kGroup, kCta = kTeams * kRowUnits<T, kGated, kStep>;
  if (units > kFp8MaxUnits) return cudaErrorInvalidValue;
  return launch_overlapped(rows_kernel<T, kGated, kStep>, dim3((unsigned)((units + kCta - 1) / kCta)), kRowThreads, 0, 0,
                           stream, static_cast<const T*>(x.ptr), x.ld, static_cast<const T*>(up.ptr), up.ld,
                           (uint32_t)rows, (uint32_t)blocks, (uint32_t)(kTeams / blocks), (uint32_t)(kTeams % blocks),
                           cols, out);
}

template <typename T, bool kGated>
cudaError_t rows_typed(Fp8In x, Fp8In up, int64_t rows, int64_t cols, Fp8Out out, cudaStream_t stream) {
  int step = step_of<T>(x.ptr, x.ld, cols);
  if (kGated) step = std::min(step, step_of<T>(up.ptr, up.ld, cols));
  if (step == 8) return rows_step<T, kGated, 8>(x, up, rows, cols, out, stream);
  if (step == 4) return rows_step<T, kGated, 4>(x, up, rows, cols, out, stream);
  return rows_step<T, kGated, 1>(x, up, rows, cols, out, stream);
}

template <typename T>
cudaError_t blocks_typed(Fp8In x, int64_t rows, int64_t cols, Fp8Out out, cudaStream_t stream) {
  const int64_t rb = (rows + kFp8Block - 1) / kFp8Block, cb = (cols + kFp8Block - 1) / kFp8Block;
  if (rb * cb > 0x7FFFFFFFLL) return cudaErrorInvalidValue;
  const T* px = static_cast<const T*>(x.ptr);
#define LLVQ_BLOCKS(S)                                                                                         \
  launch_overlapped(blocks_kernel<T, S>, dim3((unsigned)(rb * cb)), kBlockThreads, 0, 0, stream, px, x.ld, rows, cols, \
                    (uint32_t)cb, out)
  const int step = step_of<T>(px, x.ld, cols);
  return step == 8 ? LLVQ_BLOCKS(8) : step == 4 ? LLVQ_BLOCKS(4) : LLVQ_BLOCKS(1);
#undef LLVQ_BLOCKS
}

struct NormCall {
  Fp8In x, residual;
  const void* weight;
  float eps;
  int64_t rows, cols;
  void* hidden;
  int64_t ldh;
  Fp8Out out;
  cudaStream_t stream;
};

template <typename T, typename W, int kChunks, int kThreads, bool kResidual, int kStep>
cudaError_t norm_step(const NormCall& n) {
  const int64_t groups = (n.cols + kVec - 1) / kVec;
  const int threads = (int)(((groups + kChunks - 1) / kChunks + 31) / 32 * 32);
  const auto kernel = rms_norm_kernel<T, W, kChunks, kThreads, kResidual, kStep>;
  int sms = 0;
  const cudaError_t e = device_sms(&sms);
  if (e != cudaSuccess) return e;
  const int64_t resident = (int64_t)sms * std::max(1, 65536 / norm_regs(kChunks, kThreads, kStep) / threads);  // one wave
  const size_t smem = kStep == 1 ? (size_t)threads / 32 * kTurnBytes : 0;
  return launch_overlapped(kernel, dim3((unsigned)std::min(n.rows, resident)), threads, smem, 0, n.stream,
                           static_cast<const T*>(n.x.ptr), n.x.ld, static_cast<const T*>(n.residual.ptr), n.residual.ld,
                           static_cast<const W*>(n.weight), n.eps, 1.f / (float)n.cols, n.rows, n.cols,
                           static_cast<T*>(n.hidden), n.ldh, n.out);
}

template <typename T, typename W, int kChunks, int kThreads, int kStep>
cudaError_t norm_chunks(const NormCall& n) {
  return n.residual.ptr ? norm_step<T, W, kChunks, kThreads, true, kStep>(n)
                        : norm_step<T, W, kChunks, kThreads, false, kStep>(n);
}

template <typename T, typename W, int kStep>
cudaError_t norm_shape(const NormCall& n) {
  if (n.cols <= 512 * kVec) return norm_chunks<T, W, 1, 512, kStep>(n);
  if (n.cols <= 1024 * kVec) return norm_chunks<T, W, 2, 512, kStep>(n);
  return norm_chunks<T, W, 2, 1024, kStep>(n);
}

template <typename T, typename W>
cudaError_t norm_typed(const NormCall& n) {
  int step = std::min(step_of<T>(n.x.ptr, n.x.ld, n.cols), step_of<W>(n.weight, 0, n.cols));
  if (n.residual.ptr)
    step = std::min({step, step_of<T>(n.residual.ptr, n.residual.ld, n.cols), step_of<T>(n.hidden, n.ldh, n.cols)});
  if (step == 8) return norm_shape<T, W, 8>(n);
  if (step == 4) return norm_shape<T, W, 4>(n);
  // Turned loads are not ahead of their row: one chunk of more threads (2047 x
  // 16001: 40 us against 51 for two of half as many), which with a residual need
  // more registers than 1024 can have (8000 x 4097: 84 us against 99, and without
  // a residual 43 against 36).
  if (n.cols > 1024 * kVec) return norm_chunks<T, W, 2, 1024, 1>(n);
  return n.residual.ptr && n.cols <= 512 * kVec ? norm_step<T, W, 1, 512, true, 1>(n) : norm_chunks<T, W, 1, 1024, 1>(n);
}

}  // namespace

cudaError_t fp8_quantize_launch(Fp8In x, int type, int64_t rows, int64_t cols, int block_rows, Fp8Out out,
                                cudaStream_t stream) {
  if (rows <= 0 || cols <= 0) return cudaSuccess;
  if (block_rows == 1) {
    if (type == LLVQ_DT_F32) return rows_typed<float, false>(x, Fp8In{}, rows, cols, out, stream);
    if (type == LLVQ_DT_F16) return rows_typed<__half, false>(x, Fp8In{}, rows, cols, out, stream);
    return rows_typed<__nv_bfloat16, false>(x, Fp8In{}, rows, cols, out, stream);
  }
  if (type == LLVQ_DT_F32) return blocks_typed<float>(x, rows, cols, out, stream);
  if (type == LLVQ_DT_F16) return blocks_typed<__half>(x, rows, cols, out, stream);
  return blocks_typed<__nv_bfloat16>(x, rows, cols, out, stream);
}

cudaError_t fp8_swiglu_launch(Fp8In gate, Fp8In up, int type, int64_t rows, int64_t cols, Fp8Out out,
                              cudaStream_t stream) {
  if (rows <= 0 || cols <= 0) return cudaSuccess;
  if (type == LLVQ_DT_F32) return rows_typed<float, true>(gate, up, rows, cols, out, stream);
  if (type == LLVQ_DT_F16) return rows_typed<__half, true>(gate, up, rows, cols, out, stream);
  return rows_typed<__nv_bfloat16, true>(gate, up, rows, cols, out, stream);
}

cudaError_t fp8_rms_norm_launch(Fp8In x, Fp8In residual, int type, const void* weight, int weight_type, float eps,
                                int64_t rows, int64_t cols, void* hidden, int64_t ld_hidden, Fp8Out out,
                                cudaStream_t stream) {
  if (rows <= 0 || cols <= 0) return cudaSuccess;
  if (cols > kFp8NormMaxCols) return cudaErrorInvalidValue;
  const NormCall n{x, residual, weight, eps, rows, cols, hidden, ld_hidden, out, stream};
  if (type == LLVQ_DT_F32) return norm_typed<float, float>(n);
  if (type == LLVQ_DT_F16)
    return weight_type == LLVQ_DT_F32 ? norm_typed<__half, float>(n) : norm_typed<__half, __half>(n);
  return weight_type == LLVQ_DT_F32 ? norm_typed<__nv_bfloat16, float>(n)
                                    : norm_typed<__nv_bfloat16, __nv_bfloat16>(n);
}

}  // namespace llvq
