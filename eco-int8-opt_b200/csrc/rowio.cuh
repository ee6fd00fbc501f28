// 16-byte access to rows of fp32, bf16, fp16 or int8 numbers whose start has any alignment.
//
// A row is split where its first 16-byte boundary lies: `head` elements before it, `vecs`
// whole vectors, `tail` elements behind them (fewer than a vector each).  Outputs of the
// same type start at the same address modulo 16 bytes, so one split serves both.  int8 rows
// are read in groups of four from the row's start (their outputs are fp32 rows that start
// on 16 bytes): as one word where the row starts on four bytes, else byte by byte.
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
  using Raw = uint4;
  ECO_DEV static RowSplit split(const T* x, int64_t cols) {
    const int skew = (int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / (int)sizeof(T);
    RowSplit s;
    s.head = (int64_t)skew < cols ? skew : (int)cols;
    s.vecs = (cols - s.head) / E;
    s.tail = (int)(cols - s.head - s.vecs * E);
    return s;
  }
  ECO_DEV static Raw load(const T* p, int64_t v) { return __ldg(reinterpret_cast<const uint4*>(p) + v); }
  ECO_DEV static Raw load_last(const T* p, int64_t v) { return __ldcs(reinterpret_cast<const uint4*>(p) + v); }
  ECO_DEV static void unpack(const Raw& r, float (&f)[E]) {
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
  static constexpr int E = 4;
  using G = float;
  using Raw = uint32_t;
  ECO_DEV static RowSplit split(const int8_t*, int64_t cols) {
    RowSplit s;
    s.head = 0;
    s.vecs = cols / E;
    s.tail = (int)(cols - s.vecs * E);
    return s;
  }
  ECO_DEV static Raw load(const int8_t* p, int64_t v) {
    const uint8_t* q = reinterpret_cast<const uint8_t*>(p) + v * E;
    if ((reinterpret_cast<uintptr_t>(p) & 3) == 0) return __ldg(reinterpret_cast<const uint32_t*>(q));
    return (uint32_t)__ldg(q) | (uint32_t)__ldg(q + 1) << 8 | (uint32_t)__ldg(q + 2) << 16 | (uint32_t)__ldg(q + 3) << 24;
  }
  ECO_DEV static Raw load_last(const int8_t* p, int64_t v) { return load(p, v); }
  ECO_DEV static void unpack(const Raw& r, float (&f)[E]) {
#pragma unroll
    for (int i = 0; i < E; ++i) f[i] = (float)sbyte(r, i);
  }
  ECO_DEV static void store(float* p, int64_t v, const float (&f)[E]) {
    __stcs(reinterpret_cast<float4*>(p) + v, make_float4(f[0], f[1], f[2], f[3]));
  }
};
