// 16-byte access to rows of fp32, bf16, fp16 or int8 numbers whose start has any alignment.
//
// A row is split where its first 16-byte boundary lies: `head` elements before it, `vecs`
// whole vectors, `tail` elements behind them (fewer than a vector each).  Outputs of the
// same type start at the same address modulo 16 bytes, and fp32 outputs of int8 rows at four
// times that modulo 64, so one split serves both.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <type_traits>

#include "common.cuh"

ECO_DEV float to_f32(float v) { return v; }
ECO_DEV float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
ECO_DEV float to_f32(__half v) { return __half2float(v); }
ECO_DEV float to_f32(int8_t v) { return (float)v; }
template <typename T>
ECO_DEV T from_f32(float v);
template <>
ECO_DEV float from_f32<float>(float v) { return v; }
template <>
ECO_DEV __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
ECO_DEV __half from_f32<__half>(float v) { return __float2half_rn(v); }

// Eight fp32 numbers as one 32-byte store (p on 32 bytes): lanes that hold eight numbers each
// write whole sectors, where two 16-byte stores would write each sector in halves.
ECO_DEV void store_f32x8(float* p, const float* f) {
  asm volatile("st.global.cs.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(f[0]), "f"(f[1]), "f"(f[2]),
               "f"(f[3]), "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7])
               : "memory");
}

struct RowSplit {
  int head, tail;
  int64_t vecs;
  // element index of edge element e in [0, head + tail)
  ECO_DEV int64_t edge(int e, int64_t cols) const { return e < head ? e : cols - tail + (e - head); }
};

template <typename T>
struct RowIo {  // fp32, bf16, fp16
  static constexpr int E = 16 / (int)sizeof(T);
  using G = T;
  ECO_DEV static RowSplit split(const T* x, int64_t cols) {
    const int skew = (int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / (int)sizeof(T);
    RowSplit s;
    s.head = (int64_t)skew < cols ? skew : (int)cols;
    s.vecs = (cols - s.head) / E;
    s.tail = (int)(cols - s.head - s.vecs * E);
    return s;
  }
  ECO_DEV static uint4 load_last(const T* p, int64_t v) { return __ldcs(reinterpret_cast<const uint4*>(p) + v); }
  ECO_DEV static void unpack(const uint4& r, float (&f)[E]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        f[i] = __uint_as_float(w[i]);
      } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
        f[2 * i] = __uint_as_float(w[i] << 16);
        f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      } else {
        const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        f[2 * i] = t.x;
        f[2 * i + 1] = t.y;
      }
    }
  }
  ECO_DEV static float max(const uint4& r) {  // of the vector's numbers (NaN only if all are)
    if constexpr (sizeof(T) == 4) {
      return fmaxf(fmaxf(__uint_as_float(r.x), __uint_as_float(r.y)), fmaxf(__uint_as_float(r.z), __uint_as_float(r.w)));
    } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
      const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&r);
      const float2 m = __bfloat1622float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
      return fmaxf(m.x, m.y);
    } else {
      const __half2* h = reinterpret_cast<const __half2*>(&r);
      const float2 m = __half22float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
      return fmaxf(m.x, m.y);
    }
  }
  ECO_DEV static uint4 pack(const float (&f)[E]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        w[i] = __float_as_uint(f[i]);
      } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
        const __nv_bfloat162 t = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&t);
      } else {
        const __half2 t = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&t);
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  ECO_DEV static void store(T* p, int64_t v, const float (&f)[E]) { __stcs(reinterpret_cast<uint4*>(p) + v, pack(f)); }
};

template <>
struct RowIo<int8_t> {
  static constexpr int E = 16;
  using G = float;
  ECO_DEV static RowSplit split(const int8_t* x, int64_t cols) {
    const int skew = (int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15);
    RowSplit s;
    s.head = (int64_t)skew < cols ? skew : (int)cols;
    s.vecs = (cols - s.head) / E;
    s.tail = (int)(cols - s.head - s.vecs * E);
    return s;
  }
  ECO_DEV static uint4 load_last(const int8_t* p, int64_t v) { return __ldcs(reinterpret_cast<const uint4*>(p) + v); }
  ECO_DEV static void unpack(const uint4& r, float (&f)[E]) {
    // byte + 128 in the low mantissa bits of 2^23, less 2^23 + 128
    const uint32_t w[4] = {r.x ^ 0x80808080u, r.y ^ 0x80808080u, r.z ^ 0x80808080u, r.w ^ 0x80808080u};
#pragma unroll
    for (int i = 0; i < E; ++i)
      f[i] = __uint_as_float(__byte_perm(w[i / 4], 0x4B000000u, 0x7440u | (uint32_t)(i & 3))) - 8388736.0f;
  }
  ECO_DEV static float max(const uint4& r) {
    const uint32_t m = __vmaxs4(__vmaxs4(r.x, r.y), __vmaxs4(r.z, r.w));
    return (float)::max(::max(sbyte(m, 0), sbyte(m, 1)), ::max(sbyte(m, 2), sbyte(m, 3)));
  }
  ECO_DEV static void store(float* p, int64_t v, const float (&f)[E]) {
    store_f32x8(p + v * E, f);
    store_f32x8(p + v * E + 8, f + 8);
  }
};
