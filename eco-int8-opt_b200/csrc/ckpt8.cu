// Activations kept in eight bits for the backward pass.
//
// A row of `cols` numbers is put away in blocks of 128 consecutive columns (the last one may
// be shorter); a block has one fp32 scale:
//
//   amax = max |x|;  scale = amax / 127;  q = rint(x * (127 / amax))   (one fp32 rounding each)
//
// and stands for q * scale.  A block whose amax is below 2^-119 stands for zeros (127 / amax
// would leave the fp32 range near there); a block that holds an infinity or NaN stands for
// NaN throughout, so that what was not finite does not come back as something finite.
//
// A block belongs to 16 lanes of eight columns each (fp32 in the norm: a warp of four each), so
// that its maximum is a few shuffles and its bytes go out in one store per lane.  The bytes
// moved bound every kernel here; at 16384 x 8192, in us and as a share of the bandwidth of a
// copy (6.5 TB/s):
//
//           put away    bring back   gated f / b (8192 a side)   norm f / b
//   bf16    71 (0.88)   72 (0.86)    193 / 195 (0.86 / 0.85)     120 / 127 (0.86 / 0.81)
//   fp32    105 (0.98)  120 (0.86)   314 / 334 (0.92 / 0.86)     216 / 197 (0.86 / 0.94)
//
// (the norm's backward without dw; gelu in place of silu: 232 / 207 in bf16, where its arithmetic is as
// long as the copy).
#include <algorithm>
#include <cmath>

#include "abi.cuh"
#include "common.cuh"
#include "rowio.cuh"

namespace {

constexpr int kBlock = ECO_CKPT_BLOCK;  // columns per scale
constexpr int kLanes = 16;              // lanes per block, eight columns each
constexpr int kThreads = 256;
constexpr int kHalves = kThreads / kLanes;  // blocks a CTA works on at a time

// ------------------------------------------------ eight columns of a row
template <typename T, int N = 8>
struct Oct {  // N columns
  static constexpr int W = N * (int)sizeof(T) / 4;  // 32-bit words
  uint32_t w[W];
};

// Where `on`, 16 bytes; else zeros.  No branch, so that several rows' loads go out together;
// volatile: a load that counts as a pure function of its address may move in front of the
// conditions that say the address is good.
ECO_DEV uint4 load_if(const uint4* p, bool on) {
  uint4 t;
  asm volatile(
      "{ .reg .pred on; setp.ne.u32 on, %5, 0;\n"
      "mov.b32 %0, 0; mov.b32 %1, 0; mov.b32 %2, 0; mov.b32 %3, 0;\n"
      "@on ld.global.nc.v4.b32 {%0, %1, %2, %3}, [%4]; }"
      : "=&r"(t.x), "=&r"(t.y), "=&r"(t.z), "=&r"(t.w)
      : "l"(p), "r"((uint32_t)on));
  return t;
}

// Columns [c, c + n) of a row of any alignment, n in [0, N]; the others are zeros.  The 16-byte
// words that hold the columns are read and shifted into place (each word that is read holds at
// least one of them, so none lies outside the row's memory).
template <typename T, int N = 8>
ECO_DEV Oct<T, N> load8(const T* row, int c, int n) {
  constexpr int W = Oct<T, N>::W, V = W / 4;  // 32-bit words, 16-byte words
  Oct<T, N> o;
  const uintptr_t a = reinterpret_cast<uintptr_t>(row + c);
  const uint4* p = reinterpret_cast<const uint4*>(a & ~uintptr_t(15));
  const uint32_t skew = (uint32_t)a & 15;
  const int end = n > 0 ? (int)skew + n * (int)sizeof(T) : 0;  // bytes that are needed, from p on
  uint32_t w[W + 4];
#pragma unroll
  for (int v = 0; v <= V; ++v) {
    const uint4 t = load_if(p + v, 16 * v < end);
    w[4 * v] = t.x, w[4 * v + 1] = t.y, w[4 * v + 2] = t.z, w[4 * v + 3] = t.w;
  }
#pragma unroll
  for (int i = 0; i < W + 2; ++i) w[i] = skew & 8 ? w[i + 2] : w[i];
#pragma unroll
  for (int i = 0; i < W + 1; ++i) w[i] = skew & 4 ? w[i + 1] : w[i];
#pragma unroll
  for (int i = 0; i < W; ++i) {  // columns past the n-th are the row's neighbours: zeros here
    if constexpr (sizeof(T) == 4) {
      o.w[i] = i < n ? w[i] : 0u;
    } else {
      o.w[i] = __funnelshift_r(w[i], w[i + 1], (skew & 3) * 8);
      o.w[i] = 2 * i + 1 < n ? o.w[i] : (2 * i < n ? o.w[i] & 0xffffu : 0u);
    }
  }
  return o;
}

// The same, in one load where the eight columns lie on a boundary: for kernels that do not know
// of their rows.
template <typename T>
ECO_DEV Oct<T> load8_either(const T* row, int c, int n) {
  if (n < 8 || (reinterpret_cast<uintptr_t>(row + c) & 15) != 0) return load8(row, c, n);
  Oct<T> o;
#pragma unroll
  for (int v = 0; v < Oct<T>::W / 4; ++v) {
    const uint4 t = load_if(reinterpret_cast<const uint4*>(row + c) + v, true);
    o.w[4 * v] = t.x, o.w[4 * v + 1] = t.y, o.w[4 * v + 2] = t.z, o.w[4 * v + 3] = t.w;
  }
  return o;
}

template <typename T>
ECO_DEV void unpack8(const Oct<T>& o, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (sizeof(T) == 4)
      f[i] = __uint_as_float(o.w[i]);
    else if constexpr (std::is_same_v<T, __nv_bfloat16>)
      f[i] = __uint_as_float(i & 1 ? o.w[i / 2] & 0xffff0000u : o.w[i / 2] << 16);
    else
      f[i] = __half2float(__ushort_as_half((unsigned short)(o.w[i / 2] >> (16 * (i & 1)))));
  }
}

// Eight columns of an output row, past L1 (which keeps what is read again: a weight): whole where
// eight columns of the row start on a boundary of their size (its padding takes the rest of the
// last eight), else n single stores.
template <typename T>
ECO_DEV void store8(T* row, int c, int n, bool vec, const float (&f)[8]) {
  if (vec) {
    if constexpr (sizeof(T) == 4) {
      asm volatile("st.global.cg.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(row + c), "f"(f[0]), "f"(f[1]),
                   "f"(f[2]), "f"(f[3]), "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7])
                   : "memory");
    } else {
      __stcg(reinterpret_cast<uint4*>(row + c), RowIo<T>::pack(f));
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n) row[c + i] = from_f32<T>(f[i]);
}

// ------------------------------------------------ eight bits
ECO_DEV float max_nan(float a, float b) {  // NaN if either is
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
// max |x| of a block over its 16 lanes.  Without their signs, numbers order like their bits, NaN
// above infinity: an integer maximum, two 16-bit numbers at a time.
template <typename T>
ECO_DEV float block_amax(const Oct<T>& o) {
  if constexpr (sizeof(T) == 4) {
    float m = fabsf(__uint_as_float(o.w[0]));
#pragma unroll
    for (int i = 1; i < 8; ++i) m = max_nan(m, fabsf(__uint_as_float(o.w[i])));
#pragma unroll
    for (int s = 8; s > 0; s >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, s));
    return m;
  } else {
    uint32_t m = o.w[0] & 0x7fff7fffu;
#pragma unroll
    for (int i = 1; i < 4; ++i) m = __vmaxu2(m, o.w[i] & 0x7fff7fffu);
#pragma unroll
    for (int s = 8; s > 0; s >>= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, s));
    m = max(m & 0xffffu, m >> 16);
    if constexpr (std::is_same_v<T, __nv_bfloat16>) return __uint_as_float(m << 16);
    else return __half2float(__ushort_as_half((unsigned short)m));
  }
}
// Gains of N blocks of a half-warp (or warp) from their maxima, and in lane i (< N) the scale of
// block i: lane i does block i's two divisions, so that N blocks cost the divisions of one.
template <int N, int LANES = kLanes>
ECO_DEV float block_gains(const float (&amax)[N], float (&gain)[N]) {
  const int lane = threadIdx.x & (LANES - 1);
  float m = amax[0];
#pragma unroll
  for (int i = 1; i < N; ++i) m = lane == i ? amax[i] : m;
  const bool zero = m < 0x1p-119f;  // false for NaN
  const float g = zero ? 0.0f : __fdiv_rn(127.0f, m);
#pragma unroll
  for (int i = 0; i < N; ++i) gain[i] = N == 1 ? g : __shfl_sync(0xffffffffu, g, i, LANES);
  return zero ? 0.0f : (m < INFINITY ? __fdiv_rn(m, 127.0f) : __int_as_float(0x7fc00000));
}
// rint(x * gain) of eight values as bytes.  Adding 1.5 * 2^23 rounds to nearest even at the
// unit, and leaves the whole number's low byte as the sum's low byte.
ECO_DEV uint2 quant8(const float (&f)[8], float gain) {
  uint32_t b[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) b[i] = __float_as_uint(__fadd_rn(__fmul_rn(f[i], gain), 12582912.0f));
  return make_uint2(pack4(b[0], b[1], b[2], b[3]), pack4(b[4], b[5], b[6], b[7]));
}
// The bytes as floats, by the conversion unit, which has nothing else to do here.
ECO_DEV void dequant8(uint2 q, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = (float)(int8_t)((i < 4 ? q.x : q.y) >> (8 * (i & 3)));
}
// ------------------------------------------------ matrices
struct Mat {  // rows of any type
  void* p;
  int ld;
};
struct Saved {  // q [rows, ld_q] int8 (ld_q a multiple of 16), scale [rows, ld_s] fp32
  int8_t* q;
  float* scale;
  int ld_q, ld_s;
};

ECO_DEV int left8(int cols, int c) { return max(0, min(8, cols - c)); }

// Where a half-warp works: 2^l blocks of a row side by side in a CTA (up to 16), 16 / 2^l rows
// below each other; a thread keeps its eight columns and walks down the rows in groups of U,
// whose loads are all issued before the first is used (a thread has one or two 16-byte loads per
// row: alone they would not cover the memory's latency).  Both halves of a warp stay in step (the
// shuffles need all 32 lanes).  Groups of which every row exists are told apart once per group
// (`full`), for the CTA as a whole.
//   load(r) -> L for a row that exists;   use(full, L[U], first row, step)
// Lanes whose n is 0 have no columns; blocks with `live` false lie past the last.
struct Place {
  int lane, c, n, b, row, per;
  bool live;
  ECO_DEV Place(int cols, int l) {
    const int half = threadIdx.x / kLanes;
    lane = threadIdx.x & (kLanes - 1);
    b = ((int)blockIdx.x << l) + (half & ((1 << l) - 1));
    c = b * kBlock + lane * 8;
    live = b * kBlock < cols;
    n = left8(cols, c);
    row = half >> l;
    per = kHalves >> l;
  }
};
template <int U, typename L, typename Load, typename Use>
ECO_DEV void for_rows(int rows, const Place& at, Load load, Use use) {
  const int step = (int)gridDim.y * at.per;
  for (int rr = (int)blockIdx.y * at.per; rr < rows; rr += U * step) {
    const int r = rr + at.row;
    L in[U];
    if (rr + (U - 1) * step + at.per <= rows) {
#pragma unroll
      for (int u = 0; u < U; ++u) in[u] = load(r + u * step);
      use(std::true_type{}, in, r, step);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        in[u] = L{};
        if (r + u * step < rows) in[u] = load(r + u * step);
      }
      use(std::false_type{}, in, r, step);
    }
  }
}
// Eight columns of a row: WHOLE rows consist of whole groups that start on a boundary of their size.
template <typename T, bool WHOLE>
ECO_DEV Oct<T> load_cols(const Mat& x, int r, const Place& at) {
  const T* row = static_cast<const T*>(x.p) + (int64_t)r * x.ld;
  if constexpr (!WHOLE) return load8(row, at.c, at.n);
  Oct<T> o{};
  if (at.n > 0) {
    if constexpr (sizeof(T) == 4) {
      asm volatile("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                   : "=r"(o.w[0]), "=r"(o.w[1]), "=r"(o.w[2]), "=r"(o.w[3]), "=r"(o.w[4]), "=r"(o.w[5]), "=r"(o.w[6]),
                     "=r"(o.w[7])
                   : "l"(row + at.c));
    } else {
      const uint4 t = __ldg(reinterpret_cast<const uint4*>(row + at.c));
      o.w[0] = t.x, o.w[1] = t.y, o.w[2] = t.z, o.w[3] = t.w;
    }
  }
  return o;
}
template <typename T>
ECO_DEV void put_bytes(const Oct<T>& o, float gain, int8_t* q) {
  float f[8];
  unpack8(o, f);
  __stcg(reinterpret_cast<uint2*>(q), quant8(f, gain));
}

// ------------------------------------------------ put away, bring back
template <typename T, int U, bool WHOLE>
__global__ void __launch_bounds__(kThreads) pack_kernel(Mat x, int rows, int cols, Saved S, int l) {
  const Place at(cols, l);
  for_rows<U, Oct<T>>(
      rows, at, [&](int r) { return load_cols<T, WHOLE>(x, r, at); },
      [&](auto full, const Oct<T>(&o)[U], int r0, int step) {
        float amax[U], gain[U];
#pragma unroll
        for (int u = 0; u < U; ++u) amax[u] = block_amax(o[u]);
        const float scale = block_gains(amax, gain);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int r = r0 + u * step;
          if (!full && r >= rows) break;
          if (at.n > 0) put_bytes(o[u], gain[u], S.q + (int64_t)r * S.ld_q + at.c);
          if (at.lane == u && at.live) S.scale[(int64_t)r * S.ld_s + at.b] = scale;
        }
      });
}

struct Eights {
  uint2 q;
  float s;
};
ECO_DEV Eights fetch8(const Saved& S, int64_t r, int c, int n) {
  Eights e{make_uint2(0u, 0u), 0.0f};
  if (n > 0) {
    e.q = __ldcs(reinterpret_cast<const uint2*>(S.q + r * S.ld_q + c));
    e.s = __ldg(S.scale + r * S.ld_s + c / kBlock);
  }
  return e;
}
ECO_DEV void values8(const Eights& e, float (&f)[8]) {
  dequant8(e.q, f);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] *= e.s;
}

template <typename T, int U>
__global__ void __launch_bounds__(kThreads) restore_kernel(Saved S, int rows, int cols, Mat x, int l) {
  const Place at(cols, l);
  for_rows<U, Eights>(
      rows, at, [&](int r) { return fetch8(S, r, at.c, at.n); },
      [&](auto full, const Eights(&e)[U], int r0, int step) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int r = r0 + u * step;
          if (at.n == 0 || (!full && r >= rows)) break;
          float f[8];
          values8(e[u], f);
          store8(static_cast<T*>(x.p) + (int64_t)r * x.ld, at.c, at.n, true, f);
        }
      });
}

// ------------------------------------------------ gated activation
// h = act(gate) up;  d up = dh act(gate),  d gate = dh up act'(gate)
//   silu: act(g) = g s, s = 1 / (1 + e^-g);       act'(g) = s (1 + g (1 - s))
//   gelu: act(g) = g F(g), F the normal's distribution;   act'(g) = F(g) + g f(g), f its density
// The normal's distribution by the rational approximation 7.1.26 of Abramowitz and Stegun,
// Handbook of Mathematical Functions: with z = |g| / sqrt 2 and t = 1 / (1 + 0.3275911 z),
//   F(-|g|) = 1/2 (a1 t + ... + a5 t^5) exp(-z^2),  to 7.5e-8,
// whose exponential is the density's too (one exponential and one reciprocal per element for
// both; erff took as much again as all the rest).
struct Act {
  float over, dens;  // act(g) / g; gelu: the density at g
};
template <bool GELU>
ECO_DEV Act act_of(float g) {
  if (GELU) {
    const float a = fabsf(g);
    const float t = __fdividef(1.0f, fmaf(a, 0.3275911f * 0.70710678118654752f, 1.0f));
    const float e = __expf(-0.5f * g * g);
    float p = fmaf(t, 0.5f * 1.061405429f, 0.5f * -1.453152027f);
    p = fmaf(p, t, 0.5f * 1.421413741f);
    p = fmaf(p, t, 0.5f * -0.284496736f);
    p = fmaf(p, t, 0.5f * 0.254829592f);
    const float low = p * t * e;
    return Act{g < 0.0f ? low : 1.0f - low, e * 0.39894228040143268f};
  }
  return Act{__fdividef(1.0f, 1.0f + __expf(-g)), 0.0f};
}
template <bool GELU>
ECO_DEV float act_slope(float g, Act a) {
  if (GELU) return fmaf(g, a.dens, a.over);
  return a.over * fmaf(g, 1.0f - a.over, 1.0f);
}

template <typename T>
struct OctPair {
  Oct<T> a, b;
};

template <typename T, bool GELU, int U, bool WHOLE>
__global__ void __launch_bounds__(kThreads)
    gated_fwd_kernel(Mat gate, Mat up, int rows, int cols, Mat y, Saved SG, Saved SU, int l) {
  const Place at(cols, l);
  for_rows<U, OctPair<T>>(
      rows, at,
      [&](int r) { return OctPair<T>{load_cols<T, WHOLE>(gate, r, at), load_cols<T, WHOLE>(up, r, at)}; },
      [&](auto full, const OctPair<T>(&o)[U], int r0, int step) {
        float amax[2 * U], gain[2 * U], scale = 0.0f;
        if (SG.q) {
#pragma unroll
          for (int u = 0; u < U; ++u) {
            amax[2 * u] = block_amax(o[u].a);
            amax[2 * u + 1] = block_amax(o[u].b);
          }
          scale = block_gains(amax, gain);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int r = r0 + u * step;
          if (!full && r >= rows) break;
          if (SG.q) {
            if (at.n > 0) {
              put_bytes(o[u].a, gain[2 * u], SG.q + (int64_t)r * SG.ld_q + at.c);
              put_bytes(o[u].b, gain[2 * u + 1], SU.q + (int64_t)r * SU.ld_q + at.c);
            }
            if (at.lane == 2 * u && at.live) SG.scale[(int64_t)r * SG.ld_s + at.b] = scale;
            if (at.lane == 2 * u + 1 && at.live) SU.scale[(int64_t)r * SU.ld_s + at.b] = scale;
          }
          float g[8], v[8];
          unpack8(o[u].a, g);
          unpack8(o[u].b, v);
#pragma unroll
          for (int i = 0; i < 8; ++i) g[i] = g[i] * act_of<GELU>(g[i]).over * v[i];
          if (at.n > 0) store8(static_cast<T*>(y.p) + (int64_t)r * y.ld, at.c, at.n, true, g);
        }
      });
}

template <typename T>
struct GatedIn {
  Oct<T> dy;
  Eights g, u;
};

template <typename T, bool GELU, int U, bool WHOLE>
__global__ void __launch_bounds__(kThreads)
    gated_bwd_kernel(Mat dy, int rows, int cols, Saved SG, Saved SU, Mat dgate, Mat dup, bool vec_g, bool vec_u,
                     int l) {
  const Place at(cols, l);
  for_rows<U, GatedIn<T>>(
      rows, at,
      [&](int r) {
        return GatedIn<T>{load_cols<T, WHOLE>(dy, r, at), fetch8(SG, r, at.c, at.n), fetch8(SU, r, at.c, at.n)};
      },
      [&](auto full, const GatedIn<T>(&in)[U], int r0, int step) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int r = r0 + u * step;
          if (at.n == 0 || (!full && r >= rows)) break;
          float g[8], v[8], d[8];
          values8(in[u].g, g);
          values8(in[u].u, v);
          unpack8(in[u].dy, d);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const Act s = act_of<GELU>(g[i]);
            const float dg = d[i] * v[i] * act_slope<GELU>(g[i], s);
            v[i] = d[i] * g[i] * s.over;
            g[i] = dg;
          }
          store8(static_cast<T*>(dgate.p) + (int64_t)r * dgate.ld, at.c, at.n, WHOLE || (vec_g && at.n == 8), g);
          store8(static_cast<T*>(dup.p) + (int64_t)r * dup.ld, at.c, at.n, WHOLE || (vec_u && at.n == 8), v);
        }
      });
}

// ------------------------------------------------ rms norm
// y = x r w,  r = 1 / sqrt(mean x^2 + eps);  with x' = what the eight bits stand for, u = x' r:
//   dx = r (w dy - u mean(w dy u)),   dw = sum over rows of dy u.
//
// NT threads hold a row (32 columns each beyond 1024), so a row is read once; the sum is joined
// over the threads in a fixed order.  A CTA walks down its rows, and each thread copies its own
// columns of the next rows into shared memory while it works on one (cp.async: no other thread
// reads them, so no barrier belongs to the copies): the bytes in flight do not depend on how far
// the row's barrier has come.  The weight stays in shared memory as well: with this much of it
// in use L1 is too small for a weight (the backward lost a third of its time to L2's latency).
// Wider rows are read again for the second pass, and their dw sums live in the CTA's own row of
// `part`.
constexpr int kRmsThreads = 512;  // of a CTA, one per SM: 128 registers each

// A barrier of NT threads, those of row group `group` (the whole CTA has barrier 0).
template <int NT>
ECO_DEV void row_barrier(int group) {
  if constexpr (NT == 32) __syncwarp();
  else asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(NT) : "memory");
}
// Sum over the NT threads of a row; sh: NT / 32 floats of the row group's (two buffers take turns).
template <int NT>
ECO_DEV float row_sum(float v, float* sh, int group) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if constexpr (NT > 32) {
    constexpr int W = NT / 32;
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x % NT / 32] = v;
    row_barrier<NT>(group);
    v = sh[threadIdx.x % W];
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  }
  return v;
}

template <int N>
ECO_DEV void copy_async(void* dst, const void* src) {  // N bytes to shared memory
  const uint32_t d = (uint32_t)__cvta_generic_to_shared(dst);
  if constexpr (N == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d), "l"(src) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(d), "l"(src), "n"(N) : "memory");
}
ECO_DEV void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
ECO_DEV void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// A unit is 16 bytes of x (or dy): G columns, with G of the eight-bit bytes.  Unit j of thread tid is
// columns (j NT + tid) G: a warp's accesses are contiguous, and a block of 128 columns is 128 / G
// lanes of one warp.
template <typename T>
struct Unit {
  static constexpr int G = 16 / (int)sizeof(T), kLanes = kBlock / G;
  ECO_DEV static void unpack(const uint4& r, float (&f)[G]) { RowIo<T>::unpack(r, f); }
  // max |x| over the block's lanes: a whole warp's in one instruction, or half a warp's
  ECO_DEV static float amax(const uint4& r) {
    if constexpr (G == 4) {
      const uint32_t m = max(max(r.x & 0x7fffffffu, r.y & 0x7fffffffu), max(r.z & 0x7fffffffu, r.w & 0x7fffffffu));
      return __uint_as_float(__reduce_max_sync(0xffffffffu, m));
    } else {
      return block_amax(Oct<T>{{r.x, r.y, r.z, r.w}});
    }
  }
  ECO_DEV static uint4 load(const T* row, int c, int n) {  // any alignment, n of the columns
    const Oct<T, G> o = load8<T, G>(row, c, n);
    return make_uint4(o.w[0], o.w[1], o.w[2], o.w[3]);
  }
  ECO_DEV static void put_bytes(int8_t* q, const float (&f)[G], float gain) {
    uint32_t b[G];
#pragma unroll
    for (int i = 0; i < G; ++i) b[i] = __float_as_uint(__fadd_rn(__fmul_rn(f[i], gain), 12582912.0f));
    const uint32_t lo = pack4(b[0], b[1], b[2], b[3]);
    if constexpr (G == 4)
      __stcg(reinterpret_cast<uint32_t*>(q), lo);
    else
      __stcg(reinterpret_cast<uint2*>(q), make_uint2(lo, pack4(b[4], b[5], b[6], b[7])));
  }
  // byte + 128 in the low mantissa bits of 2^23, less 2^23 + 128: two short operations where a
  // conversion has a long wait
  ECO_DEV static void bytes(uint2 q, float (&f)[G]) {
    const uint32_t w[2] = {q.x ^ 0x80808080u, q.y ^ 0x80808080u};
#pragma unroll
    for (int i = 0; i < G; ++i)
      f[i] = __uint_as_float(__byte_perm(w[i / 4], 0x4B000000u, 0x7440u | (uint32_t)(i & 3))) - 8388736.0f;
  }
};
ECO_DEV int left(int cols, int c, int g) { return max(0, min(g, cols - c)); }

// The weight: nothing (ones), fp32 or x's type.
struct Weight {
  const void* p;
  bool f32;
};
template <typename T, int G>
ECO_DEV void load_weight(const Weight& w, int c, int n, float (&f)[G]) {
#pragma unroll
  for (int k = 0; k < G; ++k) f[k] = 1.0f;
  if (!w.p || n == 0) return;
  if (w.f32) {
    const float* p = static_cast<const float*>(w.p) + c;
    if (n == G && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
#pragma unroll
      for (int v = 0; v < G / 4; ++v) {
        const float4 t = __ldg(reinterpret_cast<const float4*>(p) + v);
        f[4 * v] = t.x, f[4 * v + 1] = t.y, f[4 * v + 2] = t.z, f[4 * v + 3] = t.w;
      }
      return;
    }
#pragma unroll
    for (int k = 0; k < G; ++k)
      if (k < n) f[k] = __ldg(p + k);
  } else if constexpr (sizeof(T) == 2) {
    const T* p = static_cast<const T*>(w.p) + c;
    if (n == G && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
      RowIo<T>::unpack(__ldg(reinterpret_cast<const uint4*>(p)), f);
      return;
    }
#pragma unroll
    for (int k = 0; k < G; ++k)
      if (k < n) f[k] = to_f32(p[k]);
  }
}

// Shared memory of a CTA: the weight of a row's columns in fp32, then R rows' stages for each of
// its row groups.  A stage holds what is on its way for one row: U units of all threads side by
// side; for the backward also their bytes, each block's scale and the row's rstd (copied by the
// first lane of the block or warp, read by its other lanes).
template <typename T, int NT, int U, bool BWD>
struct Stages {
  static constexpr int G = Unit<T>::G, kScales = kRmsThreads / Unit<T>::kLanes;
  static constexpr int kWeight = NT * U * G * 4;
  static constexpr int kUnit = kRmsThreads * (16 + (BWD ? G : 0)) + (BWD ? kScales * 4 : 0);
  static constexpr int kStage = U * kUnit + (BWD ? kRmsThreads / 32 * 4 : 0);
  static constexpr int kRoom = (222 * 1024 - kWeight) / kStage;
  static constexpr int R = kRoom > 4 ? 4 : kRoom;
  static constexpr int kBytes = kWeight + R * kStage;
  static_assert(R >= 1 && kUnit % 16 == 0 && kStage % 16 == 0, "a row's stage has to fit");
  char* p;
  ECO_DEV float4* weight(int j, int v) const {
    return reinterpret_cast<float4*>(p) + (j * (G / 4) + v) * NT + threadIdx.x % NT;
  }
  ECO_DEV char* unit(int s, int j) const { return p + kWeight + s * kStage + j * kUnit; }
  ECO_DEV uint4* data(int s, int j) const { return reinterpret_cast<uint4*>(unit(s, j)) + threadIdx.x; }
  ECO_DEV char* bytes(int s, int j) const { return unit(s, j) + 16 * kRmsThreads + threadIdx.x * G; }
  ECO_DEV float* scale(int s, int j) const {
    return reinterpret_cast<float*>(unit(s, j) + (16 + G) * kRmsThreads) + threadIdx.x / Unit<T>::kLanes;
  }
  ECO_DEV float* rstd(int s) const { return reinterpret_cast<float*>(unit(s, U)) + threadIdx.x / 32; }
  ECO_DEV void put_weight(int j, const float (&f)[G]) const {
#pragma unroll
    for (int v = 0; v < G / 4; ++v) *weight(j, v) = make_float4(f[4 * v], f[4 * v + 1], f[4 * v + 2], f[4 * v + 3]);
  }
  ECO_DEV void get_weight(int j, float (&f)[G]) const {
#pragma unroll
    for (int v = 0; v < G / 4; ++v) {
      const float4 t = *weight(j, v);
      f[4 * v] = t.x, f[4 * v + 1] = t.y, f[4 * v + 2] = t.z, f[4 * v + 3] = t.w;
    }
  }
};

// WHOLE: rows start on 16 bytes and consist of whole units, which are copied ahead (R rows of
// them: a unit's place is filled again as soon as it has been read); else a row is loaded when it
// is needed.
template <typename T, int NT, int U, bool WHOLE>
__global__ void __launch_bounds__(kRmsThreads, 1)
    rms_fwd_kernel(Mat x, int rows, int cols, const Weight w, float eps, Mat y, Saved S, float* rstd) {
  constexpr int GROUPS = kRmsThreads / NT;
  constexpr int G = Unit<T>::G, LB = Unit<T>::kLanes;
  using St = Stages<T, NT, U, false>;
  constexpr int R = St::R;
  extern __shared__ __align__(16) char smem[];
  __shared__ float sh[2][kRmsThreads / 32];
  const St st{smem};
  const int tid = threadIdx.x % NT, group = threadIdx.x / NT, step = (int)gridDim.x * GROUPS;
  const int lane = threadIdx.x & (LB - 1), c = tid * G;
  int r = (int)blockIdx.x * GROUPS + group;
  const float inv_cols = 1.0f / (float)cols;
  auto n_of = [&](int j) { return WHOLE ? (c + j * NT * G < cols ? G : 0) : left(cols, c + j * NT * G, G); };
  auto issue = [&](int row, int s, int j) {
    if (WHOLE && row < rows && c + j * NT * G < cols)
      copy_async<16>(st.data(s, j), static_cast<const T*>(x.p) + (int64_t)row * x.ld + c + j * NT * G);
    copies_commit();
  };
#pragma unroll
  for (int s = 0; s < R; ++s)
#pragma unroll
    for (int j = 0; j < U; ++j) issue(r + s * step, s, j);
  if (group == 0) {
#pragma unroll
    for (int j = 0; j < U; ++j) {
      float f[G];
      load_weight<T, G>(w, c + j * NT * G, n_of(j), f);
      st.put_weight(j, f);
    }
  }
  __syncthreads();
  int s = 0, par = 0;
  for (; r < rows; r += step) {
    uint4 raw[U];
    float ss = 0.0f;
#pragma unroll
    for (int j = 0; j < U; ++j) {
      raw[j] = make_uint4(0u, 0u, 0u, 0u);
      if constexpr (WHOLE) {
        copies_wait<R * U - 1>();
        if (n_of(j) > 0) raw[j] = *st.data(s, j);
        issue(r + R * step, s, j);
      } else {
        raw[j] = Unit<T>::load(static_cast<const T*>(x.p) + (int64_t)r * x.ld, c + j * NT * G, n_of(j));
      }
      float f[G];
      Unit<T>::unpack(raw[j], f);
#pragma unroll
      for (int k = 0; k < G; ++k) ss = fmaf(f[k], f[k], ss);
    }
    s = s == R - 1 ? 0 : s + 1;
    if (S.q) {  // in front of the row's barrier: it needs no sum
      float amax[U], gain[U];
#pragma unroll
      for (int j = 0; j < U; ++j) amax[j] = Unit<T>::amax(raw[j]);
      const float scale = block_gains<U, LB>(amax, gain);
      int8_t* q = S.q + (int64_t)r * S.ld_q + c;
      float* sc = S.scale + (int64_t)r * S.ld_s + c / kBlock;
#pragma unroll
      for (int j = 0; j < U; ++j) {
        float f[G];
        Unit<T>::unpack(raw[j], f);
        if (n_of(j) > 0) Unit<T>::put_bytes(q + j * NT * G, f, gain[j]);
        if (lane == j && c - G * lane + j * NT * G < cols) sc[j * (NT * G / kBlock)] = scale;
      }
    }
    ss = row_sum<NT>(ss, sh[par] + group * (NT / 32), group);
    par ^= 1;
    const float rs = rsqrtf(fmaf(ss, inv_cols, eps));
    if (tid == 0 && rstd) rstd[r] = rs;
    T* out = static_cast<T*>(y.p) + (int64_t)r * y.ld + c;
#pragma unroll
    for (int j = 0; j < U; ++j) {
      float f[G], wt[G];
      Unit<T>::unpack(raw[j], f);
      st.get_weight(j, wt);
#pragma unroll
      for (int k = 0; k < G; ++k) f[k] = f[k] * rs * wt[k];
      if (n_of(j) > 0) __stcg(reinterpret_cast<uint4*>(out + j * NT * G), RowIo<T>::pack(f));
    }
  }
}

template <typename T, int NT, int U, bool WHOLE>
__global__ void __launch_bounds__(kRmsThreads, 1)
    rms_bwd_kernel(Mat dy, int rows, int cols, const Weight w, Saved S, const float* __restrict__ rstd, Mat dx,
                   float* part, int64_t ld_part) {
  constexpr int GROUPS = kRmsThreads / NT;
  constexpr int G = Unit<T>::G, LB = Unit<T>::kLanes;
  using St = Stages<T, NT, U, true>;
  constexpr int R = St::R;
  extern __shared__ __align__(16) char smem[];
  __shared__ float sh[2][kRmsThreads / 32];
  const St st{smem};
  const int tid = threadIdx.x % NT, group = threadIdx.x / NT, step = (int)gridDim.x * GROUPS;
  const int lane = threadIdx.x & (LB - 1), c = tid * G;
  int r = (int)blockIdx.x * GROUPS + group;
  const float inv_cols = 1.0f / (float)cols;
  auto n_of = [&](int j) { return WHOLE ? (c + j * NT * G < cols ? G : 0) : left(cols, c + j * NT * G, G); };
  // What a unit's place holds of row `row`: its dy, read once; its bytes and scale, read in both
  // passes over the row (registers have no room to keep them).
  auto issue_dy = [&](int row, int s, int j) {
    if (WHOLE && row < rows && c + j * NT * G < cols)
      copy_async<16>(st.data(s, j), static_cast<const T*>(dy.p) + (int64_t)row * dy.ld + c + j * NT * G);
    copies_commit();
  };
  auto issue_bytes = [&](int row, int s, int j) {
    const int at = c + j * NT * G;
    if (WHOLE && row < rows) {
      if (at < cols) {
        copy_async<G>(st.bytes(s, j), S.q + (int64_t)row * S.ld_q + at);
        if (lane == 0) copy_async<4>(st.scale(s, j), S.scale + (int64_t)row * S.ld_s + at / kBlock);
      }
      if (j == 0 && (threadIdx.x & 31) == 0) copy_async<4>(st.rstd(s), rstd + row);
    }
    copies_commit();
  };
#pragma unroll
  for (int s = 0; s < R; ++s) {
#pragma unroll
    for (int j = 0; j < U; ++j) issue_dy(r + s * step, s, j);
#pragma unroll
    for (int j = 0; j < U; ++j) issue_bytes(r + s * step, s, j);
  }
  if (group == 0) {
#pragma unroll
    for (int j = 0; j < U; ++j) {
      float f[G];
      load_weight<T, G>(w, c + j * NT * G, n_of(j), f);
      st.put_weight(j, f);
    }
  }
  __syncthreads();
  float acc[U][G] = {};
  int s = 0, par = 0;
  for (; r < rows; r += step) {
    auto take_dy = [&](int j) {
      uint4 raw = make_uint4(0u, 0u, 0u, 0u);
      if constexpr (WHOLE) {
        // behind this unit's bytes: the rest of their row's, R - 1 rows of U + U, and this row's dy
        copies_wait<2 * U * R - U - 1>();
        if (n_of(j) > 0) raw = *st.data(s, j);
        issue_dy(r + R * step, s, j);
      } else {
        raw = Unit<T>::load(static_cast<const T*>(dy.p) + (int64_t)r * dy.ld, c + j * NT * G, n_of(j));
      }
      return raw;
    };
    auto take_bytes = [&](int j, uint2& q, float& scale) {
      q = make_uint2(0u, 0u);
      scale = 0.0f;
      if (n_of(j) == 0) return;
      if constexpr (WHOLE) {
        if constexpr (G == 8) q = *reinterpret_cast<const uint2*>(st.bytes(s, j));
        else q.x = *reinterpret_cast<const uint32_t*>(st.bytes(s, j));
        scale = *st.scale(s, j);
      } else {
        const int at = c + j * NT * G;
        const int8_t* p = S.q + (int64_t)r * S.ld_q + at;
        if constexpr (G == 8) q = __ldg(reinterpret_cast<const uint2*>(p));
        else q.x = __ldg(reinterpret_cast<const uint32_t*>(p));
        scale = __ldg(S.scale + (int64_t)r * S.ld_s + at / kBlock);
      }
    };
    // u = byte * scale * rstd: the factor, one per unit, goes where it is used once
    float dot = 0.0f, d[U][G];
    uint4 raw = take_dy(0);
    __syncwarp();  // the first lanes' copies too (scales, rstd)
    const float rs = WHOLE ? *st.rstd(s) : __ldg(rstd + r);
#pragma unroll
    for (int j = 0; j < U; ++j) {
      Unit<T>::unpack(raw, d[j]);
      uint2 q;
      float k, wt[G], u[G], part_dot = 0.0f;
      take_bytes(j, q, k);
      st.get_weight(j, wt);
      if (j + 1 < U) {
        raw = take_dy(j + 1);  // on its way while unit j is worked on
        __syncwarp();
      }
      Unit<T>::bytes(q, u);
      k *= rs;
#pragma unroll
      for (int i = 0; i < G; ++i) {
        acc[j][i] = fmaf(d[j][i] * k, u[i], acc[j][i]);
        d[j][i] *= wt[i];
        part_dot = fmaf(d[j][i], u[i], part_dot);
      }
      dot = fmaf(part_dot, k, dot);
    }
    dot = row_sum<NT>(dot, sh[par] + group * (NT / 32), group) * inv_cols;
    par ^= 1;
    T* out = static_cast<T*>(dx.p) + (int64_t)r * dx.ld + c;
    const float rd = rs * dot;
#pragma unroll
    for (int j = 0; j < U; ++j) {
      uint2 q;
      float k, u[G];
      take_bytes(j, q, k);
      Unit<T>::bytes(q, u);
      __syncwarp();  // read by all: the place is free again
      issue_bytes(r + R * step, s, j);
      k *= rd;
#pragma unroll
      for (int i = 0; i < G; ++i) d[j][i] = rs * fmaf(-u[i], k, d[j][i]);
      if (n_of(j) > 0) __stcg(reinterpret_cast<uint4*>(out + j * NT * G), RowIo<T>::pack(d[j]));
    }
    s = s == R - 1 ? 0 : s + 1;
  }
  if (part) {  // the row groups' sums to one row of them, in order
    float* mine = part + (int64_t)blockIdx.x * ld_part;
    constexpr int kSpan = U * NT * G;
    static_assert(GROUPS * kSpan * 4 <= St::kBytes, "the shared memory holds the groups' sums");
    float* joined = reinterpret_cast<float*>(smem);
    copies_wait<0>();
    __syncthreads();  // nothing there is in use
#pragma unroll
    for (int j = 0; j < U; ++j)
#pragma unroll
      for (int v = 0; v < G / 4; ++v)
        reinterpret_cast<float4*>(joined + group * kSpan + c + j * NT * G)[v] =
            make_float4(acc[j][4 * v], acc[j][4 * v + 1], acc[j][4 * v + 2], acc[j][4 * v + 3]);
    __syncthreads();
    for (int at = threadIdx.x; at < cols; at += kRmsThreads) {
      float v = joined[at];
#pragma unroll
      for (int g = 1; g < GROUPS; ++g) v += joined[g * kSpan + at];
      mine[at] = v;
    }
  }
}

// ---- rows too wide for a CTA's registers (more than 16384 columns): two passes over the row
constexpr int kWide = 512;

template <typename T>
__global__ void __launch_bounds__(kWide)
    rms_fwd_wide_kernel(Mat x, int rows, int cols, const Weight w, float eps, Mat y,
                        Saved S, float* rstd) {
  __shared__ float sh[2][kWide / 32];
  const int lane = threadIdx.x & (kLanes - 1);
  int k = 0;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x, ++k) {
    const T* row = static_cast<const T*>(x.p) + r * x.ld;
    float ss = 0.0f;
    for (int c = threadIdx.x * 8; c < cols; c += kWide * 8) {
      float f[8];
      unpack8(load8_either(row, c, left8(cols, c)), f);
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = fmaf(f[j], f[j], ss);
    }
    ss = row_sum<kWide>(ss, sh[k & 1], 0);
    const float rs = rsqrtf(ss / (float)cols + eps);
    if (threadIdx.x == 0 && rstd) rstd[r] = rs;
    for (int cc = 0; cc < cols; cc += kWide * 8) {  // every lane, for the shuffles
      const int c = cc + threadIdx.x * 8, c0 = c - 8 * lane;
      const int n = left8(cols, c);
      float f[8], wt[8];
      const Oct<T> o = load8_either(row, c, n);
      unpack8(o, f);
      if (S.q) {
        const float amax[1] = {block_amax(o)};
        float gain[1];
        const float scale = block_gains(amax, gain);
        if (n > 0) __stcg(reinterpret_cast<uint2*>(S.q + r * S.ld_q + c), quant8(f, gain[0]));
        if (lane == 0 && c0 < cols) S.scale[r * S.ld_s + c0 / kBlock] = scale;
      }
      load_weight<T, 8>(w, c, n, wt);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = f[j] * rs * wt[j];
      if (n > 0) store8(static_cast<T*>(y.p) + r * y.ld, c, n, true, f);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kWide)
    rms_bwd_wide_kernel(Mat dy, int rows, int cols, const Weight w, Saved S,
                        const float* __restrict__ rstd, Mat dx, float* part, int64_t ld_part) {
  __shared__ float sh[2][kWide / 32];
  float* mine = part ? part + blockIdx.x * ld_part : nullptr;
  int k = 0;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x, ++k) {
    const T* row = static_cast<const T*>(dy.p) + r * dy.ld;
    const float rs = rstd[r];
    float dot = 0.0f;
    for (int c = threadIdx.x * 8; c < cols; c += kWide * 8) {
      const int n = left8(cols, c);
      float d[8], u[8], wt[8];
      unpack8(load8_either(row, c, n), d);
      Eights e = fetch8(S, r, c, n);
      e.s *= rs;
      values8(e, u);
      load_weight<T, 8>(w, c, n, wt);
      if (mine) {  // a thread owns its columns of the CTA's sums: plain loads and stores, no atomics
        float4* at = reinterpret_cast<float4*>(mine + c);
        float4 s0 = make_float4(0.0f, 0.0f, 0.0f, 0.0f), s1 = s0;
        if (k) s0 = at[0], s1 = at[1];
        at[0] = make_float4(fmaf(d[0], u[0], s0.x), fmaf(d[1], u[1], s0.y), fmaf(d[2], u[2], s0.z),
                            fmaf(d[3], u[3], s0.w));
        at[1] = make_float4(fmaf(d[4], u[4], s1.x), fmaf(d[5], u[5], s1.y), fmaf(d[6], u[6], s1.z),
                            fmaf(d[7], u[7], s1.w));
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) dot = fmaf(d[j] * wt[j], u[j], dot);
    }
    dot = row_sum<kWide>(dot, sh[k & 1], 0) / (float)cols;
    for (int c = threadIdx.x * 8; c < cols; c += kWide * 8) {
      const int n = left8(cols, c);
      float d[8], u[8], wt[8];
      unpack8(load8_either(row, c, n), d);
      Eights e = fetch8(S, r, c, n);
      e.s *= rs;
      values8(e, u);
      load_weight<T, 8>(w, c, n, wt);
#pragma unroll
      for (int j = 0; j < 8; ++j) d[j] = rs * fmaf(-u[j], dot, d[j] * wt[j]);
      store8(static_cast<T*>(dx.p) + r * dx.ld, c, n, true, d);
    }
  }
}

// dw = column sums of the `n` partial rows, in double and in a fixed order: 32 columns x 32
// rows of threads per CTA, four rows' loads at a time (a thread's chain of loads is what
// takes the time).
template <typename WT>
__global__ void __launch_bounds__(1024) rms_dw_kernel(const float* __restrict__ part, int64_t n, int64_t ld_part,
                                                       int64_t cols, WT* dw) {
  __shared__ double sh[32][33];
  const int lane = threadIdx.x & 31, q = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane;
  double v = 0.0;
  if (c < cols) {
    int64_t i = q;
    for (; i + 96 < n; i += 128) {
      const float a = part[i * ld_part + c], b = part[(i + 32) * ld_part + c];
      const float d = part[(i + 64) * ld_part + c], e = part[(i + 96) * ld_part + c];
      v += (double)a + (double)b + ((double)d + (double)e);
    }
    for (; i < n; i += 32) v += part[i * ld_part + c];
  }
  sh[q][lane] = v;
  __syncthreads();
  v = sh[lane][q];  // warp q joins column q
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int64_t cq = (int64_t)blockIdx.x * 32 + q;
  if (lane == 0 && cq < cols) dw[cq] = from_f32<WT>((float)v);
}

// ------------------------------------------------ host side
// 2^l blocks side by side in a CTA: as many as leave no more than an eighth of the places empty
// (33 blocks: four side by side, nine columns of CTAs; sixteen would leave 15 of 48 places idle).
int bpr_log2_of(int64_t cols) {
  const int64_t blocks = (cols + kBlock - 1) / kBlock;
  int l = 4;
  while (l > 0 && ((-blocks & ((1 << l) - 1)) * 8 > blocks + 6)) --l;
  return l;
}
// A column of CTAs for every 2^l blocks; down the rows, as many as are resident (eight of 256
// threads per SM), each walking on.
dim3 block_grid(int64_t rows, int64_t cols, int l, int unroll) {
  const int64_t blocks = (cols + kBlock - 1) / kBlock, per = (int64_t)(kHalves >> l) * unroll;
  const int64_t gx = (blocks + (1 << l) - 1) >> l;
  const int64_t most = std::max<int64_t>(1, (int64_t)eco_num_sms() * 8 / gx);
  return dim3((unsigned)gx, (unsigned)std::min<int64_t>((rows + per - 1) / per, std::min<int64_t>(most, 65535)));
}

int check_saved(const eco_saved_i8_t* S, int64_t rows, int64_t cols, const char* who) {
  ECO_REQUIRE(S && S->q && S->scale && S->ld_q >= cols && S->ld_q <= INT32_MAX && S->ld_q % 16 == 0 &&
                  eco_aligned16(S->q) && reinterpret_cast<uintptr_t>(S->scale) % 4 == 0 &&
                  S->ld_scale >= (cols + kBlock - 1) / kBlock && S->ld_scale <= INT32_MAX,
              ECO_ERR_ARG, "%s: bad eight-bit buffers", who);
  return ECO_OK;
}
Mat mat(const void* p, int64_t ld) { return Mat{const_cast<void*>(p), (int)ld}; }
Saved saved_of(const eco_saved_i8_t* S) {
  return S ? Saved{S->q, S->scale, (int)S->ld_q, (int)S->ld_scale} : Saved{nullptr, nullptr, 0, 0};
}
int es_of(int type) { return type == ECO_F32 ? 4 : 2; }
bool good_type(int t) { return t == ECO_F32 || t == ECO_BF16 || t == ECO_F16; }
bool rows_on_16(const void* p, int64_t ld, int64_t rows, int type) {
  return eco_aligned16(p) && (rows <= 1 || ld * es_of(type) % 16 == 0);
}
// Eight columns of every row start on a boundary of their size: 32 bytes for fp32, else 16.
bool rows_on_8(const void* p, int64_t ld, int64_t rows, int type) {
  return reinterpret_cast<uintptr_t>(p) % (uintptr_t)(8 * es_of(type)) == 0 && (rows <= 1 || ld % 8 == 0);
}
// Rows of whole groups of eight columns that start on a boundary of their size.
bool whole8(const void* p, int64_t ld, int64_t rows, int64_t cols, int type) {
  return rows_on_8(p, ld, rows, type) && cols % 8 == 0;
}
int check_in(const void* p, int64_t ld, int64_t rows, int64_t cols, int type, const char* who) {
  ECO_REQUIRE(p && (rows <= 1 || (ld >= 0 && ld <= INT32_MAX)) &&
                  reinterpret_cast<uintptr_t>(p) % (uintptr_t)es_of(type) == 0,
              ECO_ERR_ARG, "%s: bad input", who);
  return ECO_OK;
}
// Outputs have rows of whole groups of eight columns that start on a boundary of their size.
int check_out(const void* p, int64_t ld, int64_t rows, int64_t cols, int type, const char* who) {
  ECO_REQUIRE(p && ld >= (cols + 7) / 8 * 8 && ld <= INT32_MAX, ECO_ERR_ARG, "%s: output rows too short", who);
  ECO_REQUIRE(rows_on_8(p, ld, 2, type), ECO_ERR_MISALIGNED, "%s: output rows do not start on eight elements", who);
  return ECO_OK;
}
int check_shape(int64_t rows, int64_t cols, int type, const char* who) {
  ECO_REQUIRE(rows >= 0 && cols > 0 && rows <= (int64_t)1 << 30 && cols <= (int64_t)1 << 28, ECO_ERR_ARG,
              "%s: bad shape", who);
  ECO_REQUIRE(good_type(type), ECO_ERR_ARG, "%s: unknown type %d", who, type);
  return ECO_OK;
}

template <typename F>
void by_float(int type, F f) {
  if (type == ECO_F32) f((float*)nullptr);
  else if (type == ECO_BF16) f((__nv_bfloat16*)nullptr);
  else f((__half*)nullptr);
}

// Threads of a row and groups of eight columns per thread: a warp up to 1024 columns, four groups
// per thread beyond; (0, 0): the two-pass kernels of wider rows.
template <typename F>
void by_width(int64_t cols, F f) {
  using std::integral_constant;
  if (cols <= 256) f(integral_constant<int, 32>{}, integral_constant<int, 1>{});
  else if (cols <= 512) f(integral_constant<int, 32>{}, integral_constant<int, 2>{});
  else if (cols <= 1024) f(integral_constant<int, 32>{}, integral_constant<int, 4>{});
  else if (cols <= 2048) f(integral_constant<int, 64>{}, integral_constant<int, 4>{});
  else if (cols <= 4096) f(integral_constant<int, 128>{}, integral_constant<int, 4>{});
  else if (cols <= 8192) f(integral_constant<int, 256>{}, integral_constant<int, 4>{});
  else if (cols <= 16384) f(integral_constant<int, 512>{}, integral_constant<int, 4>{});
  else f(integral_constant<int, 0>{}, integral_constant<int, 0>{});
}
// Rows of whole units on 16 bytes.
bool whole_rows(const void* p, int64_t ld, int64_t rows, int64_t cols, int type) {
  return rows_on_16(p, ld, rows, type) && cols * es_of(type) % 16 == 0;
}
// CTAs of the norm's kernels: what is resident (two of the two-pass kernels per SM).
int64_t rms_ctas(int64_t rows, int64_t cols) {
  int64_t n = 0;
  by_width(cols, [&](auto nt, auto) {
    constexpr int NT = decltype(nt)::value;
    const int64_t groups = NT == 0 ? 1 : kRmsThreads / (NT ? NT : 1);
    n = std::min<int64_t>((rows + groups - 1) / groups, (int64_t)eco_num_sms() * (NT == 0 ? 2 : 1));
  });
  return n;
}
// Dynamic shared memory beyond 48 KB has to be allowed once per kernel and device; the
// attribute is set at each launch that needs it (a host-side store, no synchronisation).
template <typename K>
bool allow_smem(K kernel, int bytes) {
  return bytes <= 47 * 1024 ||  // static arrays count too
         cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) == cudaSuccess;
}

}  // namespace

extern "C" int eco_ckpt_pack(const void* x, int type, int64_t rows, int64_t cols, int64_t ld,
                             const eco_saved_i8_t* saved, eco_stream_t stream) {
  if (int rc = check_shape(rows, cols, type, "eco_ckpt_pack")) return rc;
  if (rows == 0) return ECO_OK;
  if (int rc = check_in(x, ld, rows, cols, type, "eco_ckpt_pack")) return rc;
  if (int rc = check_saved(saved, rows, cols, "eco_ckpt_pack")) return rc;
  const int l = bpr_log2_of(cols);
  by_float(type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    constexpr int U = sizeof(T) == 4 ? 2 : 4;
    const auto kernel = whole8(x, ld, rows, cols, type) ? pack_kernel<T, U, true> : pack_kernel<T, U, false>;
    kernel<<<block_grid(rows, cols, l, U), kThreads, 0, eco_stream(stream)>>>(
        mat(x, ld), (int)rows, (int)cols, saved_of(saved), l);
  });
  return eco_launch_check("eco_ckpt_pack");
}

extern "C" int eco_ckpt_restore(const eco_saved_i8_t* saved, int type, int64_t rows, int64_t cols, void* x,
                                int64_t ld, eco_stream_t stream) {
  if (int rc = check_shape(rows, cols, type, "eco_ckpt_restore")) return rc;
  if (rows == 0) return ECO_OK;
  if (int rc = check_saved(saved, rows, cols, "eco_ckpt_restore")) return rc;
  if (int rc = check_out(x, ld, rows, cols, type, "eco_ckpt_restore")) return rc;
  const int l = bpr_log2_of(cols);
  by_float(type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    restore_kernel<T, 4><<<block_grid(rows, cols, l, 4), kThreads, 0, eco_stream(stream)>>>(
        saved_of(saved), (int)rows, (int)cols, mat(x, ld), l);
  });
  return eco_launch_check("eco_ckpt_restore");
}

extern "C" int eco_gated_act(const void* gate, int64_t ld_gate, const void* up, int64_t ld_up, int type, int act,
                             int64_t rows, int64_t cols, void* y, int64_t ld_y, const eco_saved_i8_t* saved_gate,
                             const eco_saved_i8_t* saved_up, eco_stream_t stream) {
  if (int rc = check_shape(rows, cols, type, "eco_gated_act")) return rc;
  ECO_REQUIRE(act == ECO_ACT_SILU || act == ECO_ACT_GELU, ECO_ERR_ARG, "eco_gated_act: unknown activation %d", act);
  ECO_REQUIRE(!saved_gate == !saved_up, ECO_ERR_ARG, "eco_gated_act: one of the two eight-bit buffers is missing");
  if (rows == 0) return ECO_OK;
  if (int rc = check_in(gate, ld_gate, rows, cols, type, "eco_gated_act")) return rc;
  if (int rc = check_in(up, ld_up, rows, cols, type, "eco_gated_act")) return rc;
  if (int rc = check_out(y, ld_y, rows, cols, type, "eco_gated_act")) return rc;
  if (saved_gate) {
    if (int rc = check_saved(saved_gate, rows, cols, "eco_gated_act")) return rc;
    if (int rc = check_saved(saved_up, rows, cols, "eco_gated_act")) return rc;
  }
  const int l = bpr_log2_of(cols);
  by_float(type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    constexpr int U = sizeof(T) == 4 ? 1 : 2;
    const dim3 grid = block_grid(rows, cols, l, U);
    const bool whole = whole8(gate, ld_gate, rows, cols, type) && whole8(up, ld_up, rows, cols, type);
    const auto kernel = act == ECO_ACT_GELU
                            ? (whole ? gated_fwd_kernel<T, true, U, true> : gated_fwd_kernel<T, true, U, false>)
                            : (whole ? gated_fwd_kernel<T, false, U, true> : gated_fwd_kernel<T, false, U, false>);
    kernel<<<grid, kThreads, 0, eco_stream(stream)>>>(mat(gate, ld_gate), mat(up, ld_up), (int)rows, (int)cols,
                                                      mat(y, ld_y), saved_of(saved_gate), saved_of(saved_up), l);
  });
  return eco_launch_check("eco_gated_act");
}

extern "C" int eco_gated_act_bwd(const void* dy, int64_t ld_dy, int type, int act, int64_t rows, int64_t cols,
                                 const eco_saved_i8_t* saved_gate, const eco_saved_i8_t* saved_up, void* dgate,
                                 int64_t ld_dgate, void* dup, int64_t ld_dup, eco_stream_t stream) {
  if (int rc = check_shape(rows, cols, type, "eco_gated_act_bwd")) return rc;
  ECO_REQUIRE(act == ECO_ACT_SILU || act == ECO_ACT_GELU, ECO_ERR_ARG, "eco_gated_act_bwd: unknown activation %d", act);
  if (rows == 0) return ECO_OK;
  if (int rc = check_in(dy, ld_dy, rows, cols, type, "eco_gated_act_bwd")) return rc;
  if (int rc = check_saved(saved_gate, rows, cols, "eco_gated_act_bwd")) return rc;
  if (int rc = check_saved(saved_up, rows, cols, "eco_gated_act_bwd")) return rc;
  ECO_REQUIRE(dgate && dup &&
                  (rows <= 1 ||
                   (ld_dgate >= cols && ld_dup >= cols && ld_dgate <= INT32_MAX && ld_dup <= INT32_MAX)),
              ECO_ERR_ARG, "eco_gated_act_bwd: bad outputs");
  // A half of one packed output has no padding of its own: the last columns, fewer than eight,
  // are stored one by one, and so is a half whose rows do not start on eight elements.
  const bool vg = rows_on_8(dgate, ld_dgate, rows, type);
  const bool vu = rows_on_8(dup, ld_dup, rows, type);
  const int l = bpr_log2_of(cols);
  by_float(type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    constexpr int U = sizeof(T) == 4 ? 1 : 2;
    const dim3 grid = block_grid(rows, cols, l, U);
    const bool whole = vg && vu && whole8(dy, ld_dy, rows, cols, type);
    const auto kernel = act == ECO_ACT_GELU
                            ? (whole ? gated_bwd_kernel<T, true, U, true> : gated_bwd_kernel<T, true, U, false>)
                            : (whole ? gated_bwd_kernel<T, false, U, true> : gated_bwd_kernel<T, false, U, false>);
    kernel<<<grid, kThreads, 0, eco_stream(stream)>>>(mat(dy, ld_dy), (int)rows, (int)cols, saved_of(saved_gate),
                                                      saved_of(saved_up), mat(dgate, ld_dgate), mat(dup, ld_dup), vg,
                                                      vu, l);
  });
  return eco_launch_check("eco_gated_act_bwd");
}

extern "C" int eco_rms_norm(const void* x, int64_t ld, int type, int64_t rows, int64_t cols, const void* w,
                            int w_type, double eps, void* y, int64_t ld_y, const eco_saved_i8_t* saved, float* rstd,
                            eco_stream_t stream) {
  if (int rc = check_shape(rows, cols, type, "eco_rms_norm")) return rc;
  ECO_REQUIRE(!w || w_type == ECO_F32 || w_type == type, ECO_ERR_ARG,
              "eco_rms_norm: the weight is fp32 or of the input's type");
  ECO_REQUIRE(std::isfinite(eps) && eps >= 0.0, ECO_ERR_ARG, "eco_rms_norm: bad eps");
  if (rows == 0) return ECO_OK;
  if (int rc = check_in(x, ld, rows, cols, type, "eco_rms_norm")) return rc;
  if (int rc = check_out(y, ld_y, rows, cols, type, "eco_rms_norm")) return rc;
  if (saved)
    if (int rc = check_saved(saved, rows, cols, "eco_rms_norm")) return rc;
  bool ok = true;
  by_float(type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    by_width(cols, [&](auto nt, auto ch) {
      constexpr int NT = decltype(nt)::value, CH = decltype(ch)::value;
      const unsigned grid = (unsigned)rms_ctas(rows, cols);
      const Mat xi = mat(x, ld), yo = mat(y, ld_y);
      const Weight wt{w, w_type == ECO_F32};
      if constexpr (NT == 0) {
        rms_fwd_wide_kernel<T><<<grid, kWide, 0, eco_stream(stream)>>>(xi, (int)rows, (int)cols, wt, (float)eps, yo,
                                                                       saved_of(saved), rstd);
      } else {
        constexpr int U = CH * 8 / Unit<T>::G, smem = Stages<T, NT, U, false>::kBytes;
        const auto kernel = whole_rows(x, ld, rows, cols, type) ? rms_fwd_kernel<T, NT, U, true>
                                                                : rms_fwd_kernel<T, NT, U, false>;
        ok = allow_smem(kernel, smem);
        if (ok)
          kernel<<<grid, kRmsThreads, smem, eco_stream(stream)>>>(xi, (int)rows, (int)cols, wt, (float)eps, yo,
                                                              saved_of(saved), rstd);
      }
    });
  });
  if (!ok) return eco_fail(ECO_ERR_LAUNCH, "eco_rms_norm: %s", cudaGetErrorString(cudaGetLastError()));
  return eco_launch_check("eco_rms_norm");
}

extern "C" int64_t eco_rms_norm_bwd_scratch(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0) return 0;
  return rms_ctas(rows, cols) * ((cols + 7) / 8 * 8);
}

extern "C" int eco_rms_norm_bwd(const void* dy, int64_t ld_dy, int type, int64_t rows, int64_t cols, const void* w,
                                int w_type, const eco_saved_i8_t* saved, const float* rstd, void* dx, int64_t ld_dx,
                                void* dw, float* scratch, int64_t scratch_len, eco_stream_t stream) {
  if (int rc = check_shape(rows, cols, type, "eco_rms_norm_bwd")) return rc;
  ECO_REQUIRE(!w || w_type == ECO_F32 || w_type == type, ECO_ERR_ARG,
              "eco_rms_norm_bwd: the weight is fp32 or of the input's type");
  ECO_REQUIRE(!dw || w, ECO_ERR_ARG, "eco_rms_norm_bwd: a weight gradient needs the weight");
  cudaStream_t s = eco_stream(stream);
  if (rows == 0) {
    if (dw && cudaMemsetAsync(dw, 0, (size_t)cols * es_of(w_type), s) != cudaSuccess)
      return eco_launch_check("eco_rms_norm_bwd");
    return ECO_OK;
  }
  if (int rc = check_in(dy, ld_dy, rows, cols, type, "eco_rms_norm_bwd")) return rc;
  if (int rc = check_saved(saved, rows, cols, "eco_rms_norm_bwd")) return rc;
  if (int rc = check_out(dx, ld_dx, rows, cols, type, "eco_rms_norm_bwd")) return rc;
  ECO_REQUIRE(rstd && reinterpret_cast<uintptr_t>(rstd) % 4 == 0, ECO_ERR_ARG, "eco_rms_norm_bwd: bad rstd");
  const int64_t ctas = rms_ctas(rows, cols), ld_part = (cols + 7) / 8 * 8;
  ECO_REQUIRE(!dw || (scratch && eco_aligned16(scratch) && scratch_len >= ctas * ld_part), ECO_ERR_ARG,
              "eco_rms_norm_bwd: scratch too small (eco_rms_norm_bwd_scratch)");
  bool ok = true;
  by_float(type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    by_width(cols, [&](auto nt, auto ch) {
      constexpr int NT = decltype(nt)::value, CH = decltype(ch)::value;
      const unsigned grid = (unsigned)ctas;
      const Mat d = mat(dy, ld_dy), o = mat(dx, ld_dx);
      float* part = dw ? scratch : nullptr;
      const Weight wt{w, w_type == ECO_F32};
      if constexpr (NT == 0) {
        rms_bwd_wide_kernel<T><<<grid, kWide, 0, s>>>(d, (int)rows, (int)cols, wt, saved_of(saved), rstd, o, part,
                                                           ld_part);
      } else {
        constexpr int U = CH * 8 / Unit<T>::G, smem = Stages<T, NT, U, true>::kBytes;
        const auto kernel = whole_rows(dy, ld_dy, rows, cols, type) ? rms_bwd_kernel<T, NT, U, true>
                                                                    : rms_bwd_kernel<T, NT, U, false>;
        ok = allow_smem(kernel, smem);
        if (ok)
          kernel<<<grid, kRmsThreads, smem, s>>>(d, (int)rows, (int)cols, wt, saved_of(saved), rstd, o, part, ld_part);
      }
    });
  });
  if (!ok) return eco_fail(ECO_ERR_LAUNCH, "eco_rms_norm_bwd: %s", cudaGetErrorString(cudaGetLastError()));
  if (dw)
    by_float(w_type, [&](auto* t) {
      using WT = std::remove_pointer_t<decltype(t)>;
      rms_dw_kernel<WT><<<(unsigned)((cols + 31) / 32), 1024, 0, s>>>(scratch, ctas, ld_part, cols,
                                                                     static_cast<WT*>(dw));
    });
  return eco_launch_check("eco_rms_norm_bwd");
}
