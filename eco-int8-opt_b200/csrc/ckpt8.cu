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
// Every kernel here gives a block to 16 lanes, eight columns each: the maximum is four
// shuffles, the eight bytes one 8-byte store, and the bytes moved are the bound.
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
template <typename T>
struct Oct {
  static constexpr int W = 2 * (int)sizeof(T);  // 32-bit words
  uint32_t w[W];
};

// Columns [c, c + n) of a row, n in [0, 8]; the others are zeros.  A row that does not start
// on 16 bytes (32 for fp32) is read by the 16-byte words that hold its columns, shifted into
// place (each word that is read holds at least one of them, so none lies outside the row's memory).
template <typename T>
ECO_DEV Oct<T> load8(const T* row, int64_t c, int n) {
  constexpr int W = Oct<T>::W, V = W / 4;  // 32-bit words, 16-byte words
  Oct<T> o;
  const uintptr_t a = reinterpret_cast<uintptr_t>(row + c);
  if (n == 8 && (a & (16 * V - 1)) == 0) {
    if constexpr (V == 2) {
      asm("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
          : "=r"(o.w[0]), "=r"(o.w[1]), "=r"(o.w[2]), "=r"(o.w[3]), "=r"(o.w[4]), "=r"(o.w[5]), "=r"(o.w[6]), "=r"(o.w[7])
          : "l"(row + c));
    } else {
      const uint4 t = __ldg(reinterpret_cast<const uint4*>(row + c));
      o.w[0] = t.x, o.w[1] = t.y, o.w[2] = t.z, o.w[3] = t.w;
    }
    return o;
  }
  const uint4* p = reinterpret_cast<const uint4*>(a & ~uintptr_t(15));
  const uint32_t skew = (uint32_t)a & 15;
  const int end = n > 0 ? (int)skew + n * (int)sizeof(T) : 0;  // bytes that are needed, from p on
  uint32_t w[W + 4];
#pragma unroll
  for (int v = 0; v <= V; ++v) {
    uint4 t = make_uint4(0u, 0u, 0u, 0u);
    if (16 * v < end) t = __ldg(p + v);
    w[4 * v] = t.x, w[4 * v + 1] = t.y, w[4 * v + 2] = t.z, w[4 * v + 3] = t.w;
  }
  if (skew & 8) {
#pragma unroll
    for (int i = 0; i < W + 2; ++i) w[i] = w[i + 2];
  }
  if (skew & 4) {
#pragma unroll
    for (int i = 0; i < W + 1; ++i) w[i] = w[i + 1];
  }
  const uint32_t bits = (skew & 3) * 8;
#pragma unroll
  for (int i = 0; i < W; ++i) {  // columns past the n-th are the row's neighbours: zeros here
    o.w[i] = __funnelshift_r(w[i], w[i + 1], bits);
    if constexpr (sizeof(T) == 4)
      o.w[i] = i < n ? o.w[i] : 0u;
    else
      o.w[i] = 2 * i + 1 < n ? o.w[i] : (2 * i < n ? o.w[i] & 0xffffu : 0u);
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

// Eight columns of an output row: whole where eight columns of the row start on a boundary of
// their size (its padding takes the rest of the last eight), else n single stores.
template <typename T>
ECO_DEV void store8(T* row, int64_t c, int n, bool vec, const float (&f)[8]) {
  if (vec) {
    if constexpr (sizeof(T) == 4) {
      asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(row + c), "f"(f[0]), "f"(f[1]),
                   "f"(f[2]), "f"(f[3]), "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7])
                   : "memory");
    } else {
      *reinterpret_cast<uint4*>(row + c) = RowIo<T>::pack(f);
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
// Gains of N blocks of a half-warp from their maxima, and in lane i (< N) the scale of block i:
// lane i does block i's two divisions, so that N blocks cost the divisions of one.
template <int N>
ECO_DEV float block_gains(const float (&amax)[N], float (&gain)[N]) {
  const int lane = threadIdx.x & (kLanes - 1);
  float m = amax[0];
#pragma unroll
  for (int i = 1; i < N; ++i) m = lane == i ? amax[i] : m;
  const bool zero = m < 0x1p-119f;  // false for NaN
  const float g = zero ? 0.0f : __fdiv_rn(127.0f, m);
#pragma unroll
  for (int i = 0; i < N; ++i) gain[i] = N == 1 ? g : __shfl_sync(0xffffffffu, g, i, kLanes);
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
// The bytes as floats: byte + 128 in the low mantissa bits of 2^23, less 2^23 + 128.
ECO_DEV void dequant8(uint2 q, float (&f)[8]) {
  const uint32_t w[2] = {q.x ^ 0x80808080u, q.y ^ 0x80808080u};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    f[i] = __uint_as_float(__byte_perm(w[i / 4], 0x4B000000u, 0x7440u | (uint32_t)(i & 3))) - 8388736.0f;
}
// ------------------------------------------------ matrices
struct Mat {  // rows of any type; two leading dimensions collapse to one
  void* p;
  int64_t ld;
};
struct Saved {  // q [rows, ld_q] int8 (ld_q a multiple of 16), scale [rows, ld_s] fp32
  int8_t* q;
  float* scale;
  int64_t ld_q, ld_s;
};

ECO_DEV int left8(int64_t cols, int64_t c) { return cols - c >= 8 ? 8 : (cols > c ? (int)(cols - c) : 0); }

// Where a half-warp works: blocks of one row side by side, rows below each other.  bpr
// (blocks of a row in a CTA, a power of two up to 16) times rows in a CTA = 16.
struct Tile {
  int64_t row0, row_step;
  int64_t b0, b_step, blocks;
  int lane;
  ECO_DEV Tile(int64_t cols, int bpr_log2) {
    const int half = threadIdx.x / kLanes;
    lane = threadIdx.x & (kLanes - 1);
    blocks = (cols + kBlock - 1) / kBlock;
    const int rows = kHalves >> bpr_log2;
    row0 = (int64_t)blockIdx.y * rows + (half >> bpr_log2);
    row_step = (int64_t)gridDim.y * rows;
    b0 = ((int64_t)blockIdx.x << bpr_log2) + (half & ((1 << bpr_log2) - 1));
    b_step = (int64_t)gridDim.x << bpr_log2;
  }
};
// Loops over (row, block) in groups of U rows, whose loads are all issued before the first is
// used (a thread has one or two 16-byte loads per row: alone they would not cover the memory's
// latency).  Both halves of a warp stay in step (the shuffles need all 32 lanes): lanes past the
// last row or column get n = 0 columns, blocks past the last row or block `live` = false.
// load(r, c, n) -> L;  use(L[U], r[U], n[U], live[U], b, c).
template <int U, typename L, typename Load, typename Use>
ECO_DEV void for_blocks(int64_t rows, int64_t cols, int bpr_log2, Load load, Use use) {
  const Tile t(cols, bpr_log2);
  const int64_t first = (int64_t)blockIdx.y * (kHalves >> bpr_log2), firstb = (int64_t)blockIdx.x << bpr_log2;
  for (int64_t r0 = t.row0, rr = first; rr < rows; r0 += U * t.row_step, rr += U * t.row_step)
    for (int64_t b = t.b0, bb = firstb; bb < t.blocks; b += t.b_step, bb += t.b_step) {
      const int64_t c = b * kBlock + t.lane * 8;
      L l[U];
      int64_t r[U];
      int n[U];
      bool live[U];
      const int most = b < t.blocks ? left8(cols, c) : 0;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        r[u] = r0 + u * t.row_step;
        live[u] = r[u] < rows && b < t.blocks;
        n[u] = live[u] ? most : 0;
        if (!live[u]) r[u] = 0;
        l[u] = load(r[u], c, n[u]);
      }
      use(l, r, n, live, b, c);
    }
}

// ------------------------------------------------ put away, bring back
template <typename T, int U>
__global__ void __launch_bounds__(kThreads) pack_kernel(Mat x, int64_t rows, int64_t cols, Saved S, int bpr_log2) {
  for_blocks<U, Oct<T>>(
      rows, cols, bpr_log2,
      [&](int64_t r, int64_t c, int n) { return load8(static_cast<const T*>(x.p) + r * x.ld, c, n); },
      [&](const Oct<T>(&o)[U], const int64_t(&r)[U], const int(&n)[U], const bool(&live)[U], int64_t b, int64_t c) {
        float f[8], amax[U], gain[U];
#pragma unroll
        for (int u = 0; u < U; ++u) amax[u] = block_amax(o[u]);
        const float scale = block_gains(amax, gain);
        const int lane = threadIdx.x & (kLanes - 1);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          unpack8(o[u], f);
          if (n[u] > 0) __stcs(reinterpret_cast<uint2*>(S.q + r[u] * S.ld_q + c), quant8(f, gain[u]));
          if (lane == u && live[u]) S.scale[r[u] * S.ld_s + b] = scale;
        }
      });
}

struct Eights {
  uint2 q;
  float s;
};
ECO_DEV Eights fetch8(const Saved& S, int64_t r, int64_t c, int n) {
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
__global__ void __launch_bounds__(kThreads) restore_kernel(Saved S, int64_t rows, int64_t cols, Mat x, int bpr_log2) {
  for_blocks<U, Eights>(
      rows, cols, bpr_log2, [&](int64_t r, int64_t c, int n) { return fetch8(S, r, c, n); },
      [&](const Eights(&e)[U], const int64_t(&r)[U], const int(&n)[U], const bool(&live)[U], int64_t b, int64_t c) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          float f[8];
          values8(e[u], f);
          if (n[u] > 0) store8(static_cast<T*>(x.p) + r[u] * x.ld, c, n[u], true, f);
        }
      });
}

// ------------------------------------------------ gated activation
// h = act(gate) up;  d up = dh act(gate),  d gate = dh up act'(gate)
//   silu: act(g) = g s, s = 1 / (1 + e^-g);       act'(g) = s (1 + g (1 - s))
//   gelu: act(g) = g F(g), F the normal's distribution;   act'(g) = F(g) + g f(g), f its density
template <bool GELU>
ECO_DEV float act_over_input(float g) {
  if (GELU) return 0.5f * (1.0f + erff(g * 0.70710678118654752f));
  return __fdividef(1.0f, 1.0f + __expf(-g));
}
template <bool GELU>
ECO_DEV float act_slope(float g, float s) {
  if (GELU) return fmaf(g * 0.39894228040143268f, __expf(-0.5f * g * g), s);
  return s * fmaf(g, 1.0f - s, 1.0f);
}

template <typename T>
struct OctPair {
  Oct<T> a, b;
};

template <typename T, bool GELU, int U>
__global__ void __launch_bounds__(kThreads)
    gated_fwd_kernel(Mat gate, Mat up, int64_t rows, int64_t cols, Mat y, Saved SG, Saved SU, int bpr_log2) {
  for_blocks<U, OctPair<T>>(
      rows, cols, bpr_log2,
      [&](int64_t r, int64_t c, int n) {
        return OctPair<T>{load8(static_cast<const T*>(gate.p) + r * gate.ld, c, n),
                          load8(static_cast<const T*>(up.p) + r * up.ld, c, n)};
      },
      [&](const OctPair<T>(&o)[U], const int64_t(&r)[U], const int(&n)[U], const bool(&live)[U], int64_t b, int64_t c) {
        const int lane = threadIdx.x & (kLanes - 1);
        if (SG.q) {
          float f[8], amax[2 * U], gain[2 * U];
#pragma unroll
          for (int u = 0; u < U; ++u) {
            amax[2 * u] = block_amax(o[u].a);
            amax[2 * u + 1] = block_amax(o[u].b);
          }
          const float scale = block_gains(amax, gain);
#pragma unroll
          for (int u = 0; u < U; ++u) {
            if (n[u] > 0) {
              unpack8(o[u].a, f);
              __stcs(reinterpret_cast<uint2*>(SG.q + r[u] * SG.ld_q + c), quant8(f, gain[2 * u]));
              unpack8(o[u].b, f);
              __stcs(reinterpret_cast<uint2*>(SU.q + r[u] * SU.ld_q + c), quant8(f, gain[2 * u + 1]));
            }
            if (lane == 2 * u && live[u]) SG.scale[r[u] * SG.ld_s + b] = scale;
            if (lane == 2 * u + 1 && live[u]) SU.scale[r[u] * SU.ld_s + b] = scale;
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          float g[8], v[8];
          unpack8(o[u].a, g);
          unpack8(o[u].b, v);
#pragma unroll
          for (int i = 0; i < 8; ++i) g[i] = g[i] * act_over_input<GELU>(g[i]) * v[i];
          if (n[u] > 0) store8(static_cast<T*>(y.p) + r[u] * y.ld, c, n[u], true, g);
        }
      });
}

template <typename T>
struct GatedIn {
  Oct<T> dy;
  Eights g, u;
};

template <typename T, bool GELU, int U>
__global__ void __launch_bounds__(kThreads)
    gated_bwd_kernel(Mat dy, int64_t rows, int64_t cols, Saved SG, Saved SU, Mat dgate, Mat dup, bool vec_g,
                     bool vec_u, int bpr_log2) {
  for_blocks<U, GatedIn<T>>(
      rows, cols, bpr_log2,
      [&](int64_t r, int64_t c, int n) {
        return GatedIn<T>{load8(static_cast<const T*>(dy.p) + r * dy.ld, c, n), fetch8(SG, r, c, n),
                          fetch8(SU, r, c, n)};
      },
      [&](const GatedIn<T>(&in)[U], const int64_t(&r)[U], const int(&n)[U], const bool(&live)[U], int64_t b, int64_t c) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          float g[8], v[8], d[8];
          values8(in[u].g, g);
          values8(in[u].u, v);
          unpack8(in[u].dy, d);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float s = act_over_input<GELU>(g[i]);
            const float dg = d[i] * v[i] * act_slope<GELU>(g[i], s);
            v[i] = d[i] * g[i] * s;
            g[i] = dg;
          }
          if (n[u] > 0) {
            store8(static_cast<T*>(dgate.p) + r[u] * dgate.ld, c, n[u], vec_g && n[u] == 8, g);
            store8(static_cast<T*>(dup.p) + r[u] * dup.ld, c, n[u], vec_u && n[u] == 8, v);
          }
        }
      });
}

// ------------------------------------------------ rms norm
// y = x r w,  r = 1 / sqrt(mean x^2 + eps);  with x' = what the eight bits stand for, u = x' r:
//   dx = r (w dy - u mean(w dy u)),   dw = sum over rows of dy u.
//
// NT threads hold a row, 16 columns each, so a row is read once; the sum is joined over the
// threads in a fixed order, with one barrier a row.  A CTA walks down its rows, and each thread
// copies its own columns of the next rows (Stage::kAhead) into shared memory while it works on one
// (cp.async: no other thread reads them, so no barrier belongs to the copies): the bytes in
// flight do not depend on how far the row's barrier has come.  Rows that do not start on 16
// bytes are loaded when they are needed.  Wider rows are read again for the second pass, and
// their dw sums live in the CTA's own row of `part`.
constexpr int kCh = 2;      // groups of eight columns per thread

template <int NT>
ECO_DEV float row_sum(float v, float* sh) {  // sh: this row's buffer (two take turns)
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (NT > 32) {
    constexpr int W = NT / 32;
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    v = sh[threadIdx.x % W];
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  }
  return v;
}

// cp.async of `bytes` (0 .. N; the rest is zeros) to N bytes of shared memory.
template <int N>
ECO_DEV void copy_async(void* dst, const void* src, int bytes) {
  const uint32_t d = (uint32_t)__cvta_generic_to_shared(dst);
  if constexpr (N == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d), "l"(src), "r"(bytes) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(d), "l"(src), "n"(N), "r"(bytes) : "memory");
}
ECO_DEV void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
ECO_DEV void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// One thread's columns of a row on their way: kCh groups of T (16-byte pieces, a piece of all
// threads side by side), and for the backward the bytes, scales and the row's rstd.
template <typename T, bool BWD>
struct Stage {
  static constexpr int V = Oct<T>::W / 4;
  static constexpr int kBytes = kCh * 16 * V + (BWD ? kCh * 12 + 4 : 0);  // per thread
  // Rows on their way besides the one in work: what 1024 threads' stages leave room for.
  static constexpr int kAhead = 200 * 1024 / (kBytes * 1024) - 1 > 3 ? 3 : 200 * 1024 / (kBytes * 1024) - 1;
  ECO_DEV static uint4* piece(char* st, int threads, int i, int v) {
    return reinterpret_cast<uint4*>(st) + (i * V + v) * threads + threadIdx.x;
  }
  ECO_DEV static uint2* bytes(char* st, int threads, int i) {
    return reinterpret_cast<uint2*>(st + kCh * 16 * V * threads) + i * threads + threadIdx.x;
  }
  ECO_DEV static float* word(char* st, int threads, int i) {  // scales, then rstd
    return reinterpret_cast<float*>(st + kCh * (16 * V + 8) * threads) + i * threads + threadIdx.x;
  }
};

// The weight of a thread's columns (ones without a weight, zeros past the end).
template <typename T>
ECO_DEV void load_weight(const void* w, bool w_f32, int64_t cols, int64_t c, float (&f)[8]) {
  const int n = left8(cols, c);
  if (!w) {
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = 1.0f;
  } else if (w_f32) {
    unpack8(load8(static_cast<const float*>(w), c, n), f);
  } else {
    unpack8(load8(static_cast<const T*>(w), c, n), f);
  }
}

template <typename T, int NT>
__global__ void __launch_bounds__(NT == 32 ? kThreads : NT, NT == 32 ? 1024 / kThreads : 1024 / NT)
    rms_fwd_kernel(Mat x, int64_t rows, int64_t cols, const void* __restrict__ w, bool w_f32, float eps, Mat y,
                   Saved S, float* rstd, bool async) {
  extern __shared__ __align__(16) char stages[];
  __shared__ float sh[2][NT / 32];
  using St = Stage<T, false>;
  constexpr int THREADS = NT == 32 ? kThreads : NT, RPC = THREADS / NT;
  constexpr int kStage = St::kBytes * THREADS, kAhead = St::kAhead;
  const int tid = threadIdx.x % NT;
  const int64_t step = (int64_t)gridDim.x * RPC;
  int64_t r = (int64_t)blockIdx.x * RPC + threadIdx.x / NT;
  auto column = [&](int i) { return ((int64_t)i * NT + tid) * 8; };
  auto issue = [&](int64_t row, int slot) {
    if (async && row < rows) {
      const T* p = static_cast<const T*>(x.p) + row * x.ld;
#pragma unroll
      for (int i = 0; i < kCh; ++i) {
        const int n = left8(cols, column(i)) * (int)sizeof(T);
#pragma unroll
        for (int v = 0; v < St::V; ++v) {
          const int b = n - 16 * v < 0 ? 0 : (n - 16 * v > 16 ? 16 : n - 16 * v);
          copy_async<16>(St::piece(stages + slot * kStage, THREADS, i, v), b > 0 ? p + column(i) + 4 * v : p, b);
        }
      }
    }
    copies_commit();
  };
  for (int d = 0; d < kAhead; ++d) issue(r + d * step, d);
  float wt[kCh][8];
#pragma unroll
  for (int i = 0; i < kCh; ++i) load_weight<T>(w, w_f32, cols, column(i), wt[i]);
  for (int k = 0; r < rows; ++k, r += step) {
    issue(r + kAhead * step, (k + kAhead) % (kAhead + 1));
    Oct<T> o[kCh];
    if (async) {
      copies_wait<kAhead>();
      char* st = stages + (k % (kAhead + 1)) * kStage;
#pragma unroll
      for (int i = 0; i < kCh; ++i)
#pragma unroll
        for (int v = 0; v < St::V; ++v) {
          const uint4 q = *St::piece(st, THREADS, i, v);
          o[i].w[4 * v] = q.x, o[i].w[4 * v + 1] = q.y, o[i].w[4 * v + 2] = q.z, o[i].w[4 * v + 3] = q.w;
        }
    } else {
#pragma unroll
      for (int i = 0; i < kCh; ++i)
        o[i] = load8(static_cast<const T*>(x.p) + r * x.ld, column(i), left8(cols, column(i)));
    }
    float ss = 0.0f, f[kCh][8];
#pragma unroll
    for (int i = 0; i < kCh; ++i) {
      unpack8(o[i], f[i]);
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = fmaf(f[i][j], f[i][j], ss);
    }
    ss = row_sum<NT>(ss, sh[k & 1]);
    const float rs = rsqrtf(ss / (float)cols + eps);
    if (tid == 0 && rstd) rstd[r] = rs;
    if (S.q) {
      float amax[kCh], gain[kCh];
#pragma unroll
      for (int i = 0; i < kCh; ++i) amax[i] = block_amax(o[i]);
      const float scale = block_gains(amax, gain);
      const int lane = threadIdx.x & (kLanes - 1);
#pragma unroll
      for (int i = 0; i < kCh; ++i) {
        const int64_t c = column(i), c0 = c - 8 * lane;  // the block's first column
        if (c < cols) __stcs(reinterpret_cast<uint2*>(S.q + r * S.ld_q + c), quant8(f[i], gain[i]));
        if (lane == i && c0 < cols) S.scale[r * S.ld_s + c0 / kBlock] = scale;
      }
    }
#pragma unroll
    for (int i = 0; i < kCh; ++i) {
#pragma unroll
      for (int j = 0; j < 8; ++j) f[i][j] = f[i][j] * rs * wt[i][j];
      const int n = left8(cols, column(i));
      if (n > 0) store8(static_cast<T*>(y.p) + r * y.ld, column(i), n, true, f[i]);
    }
  }
}

template <typename T, int NT>
__global__ void __launch_bounds__(NT == 32 ? kThreads : NT, NT == 32 ? 1024 / kThreads : 1024 / NT)
    rms_bwd_kernel(Mat dy, int64_t rows, int64_t cols, const void* __restrict__ w, bool w_f32, Saved S,
                   const float* __restrict__ rstd, Mat dx, float* part, int64_t ld_part, bool async) {
  extern __shared__ __align__(16) char stages[];
  __shared__ float sh[2][NT / 32];
  using St = Stage<T, true>;
  constexpr int THREADS = NT == 32 ? kThreads : NT, RPC = THREADS / NT;
  constexpr int kStage = St::kBytes * THREADS, kAhead = St::kAhead;
  const int tid = threadIdx.x % NT;
  const int64_t step = (int64_t)gridDim.x * RPC;
  int64_t r = (int64_t)blockIdx.x * RPC + threadIdx.x / NT;
  auto column = [&](int i) { return ((int64_t)i * NT + tid) * 8; };
  auto issue = [&](int64_t row, int slot) {
    if (async && row < rows) {
      char* st = stages + slot * kStage;
      const T* p = static_cast<const T*>(dy.p) + row * dy.ld;
      const int8_t* q = S.q + row * S.ld_q;
      const float* sc = S.scale + row * S.ld_s;
#pragma unroll
      for (int i = 0; i < kCh; ++i) {
        const int64_t c = column(i);
        const int n = left8(cols, c) * (int)sizeof(T);
#pragma unroll
        for (int v = 0; v < St::V; ++v) {
          const int b = n - 16 * v < 0 ? 0 : (n - 16 * v > 16 ? 16 : n - 16 * v);
          copy_async<16>(St::piece(st, THREADS, i, v), b > 0 ? p + c + 4 * v : p, b);
        }
        copy_async<8>(St::bytes(st, THREADS, i), n > 0 ? q + c : q, n > 0 ? 8 : 0);
        copy_async<4>(St::word(st, THREADS, i), n > 0 ? sc + c / kBlock : sc, n > 0 ? 4 : 0);
      }
      copy_async<4>(St::word(st, THREADS, kCh), rstd + row, 4);
    }
    copies_commit();
  };
  for (int d = 0; d < kAhead; ++d) issue(r + d * step, d);
  float acc[kCh][8] = {};
  for (int k = 0; r < rows; ++k, r += step) {
    issue(r + kAhead * step, (k + kAhead) % (kAhead + 1));
    Oct<T> o[kCh];
    Eights e[kCh];
    float rs;
    if (async) {
      copies_wait<kAhead>();
      char* st = stages + (k % (kAhead + 1)) * kStage;
#pragma unroll
      for (int i = 0; i < kCh; ++i) {
#pragma unroll
        for (int v = 0; v < St::V; ++v) {
          const uint4 q = *St::piece(st, THREADS, i, v);
          o[i].w[4 * v] = q.x, o[i].w[4 * v + 1] = q.y, o[i].w[4 * v + 2] = q.z, o[i].w[4 * v + 3] = q.w;
        }
        e[i].q = *St::bytes(st, THREADS, i);
        e[i].s = *St::word(st, THREADS, i);
      }
      rs = *St::word(st, THREADS, kCh);
    } else {
#pragma unroll
      for (int i = 0; i < kCh; ++i) {
        const int n = left8(cols, column(i));
        o[i] = load8(static_cast<const T*>(dy.p) + r * dy.ld, column(i), n);
        e[i] = fetch8(S, r, column(i), n);
      }
      rs = rstd[r];
    }
    float dot = 0.0f, d[kCh][8], u[kCh][8];
#pragma unroll
    for (int i = 0; i < kCh; ++i) {
      float wt[8];
      load_weight<T>(w, w_f32, cols, column(i), wt);  // from L1: registers hold the sums
      unpack8(o[i], d[i]);
      e[i].s *= rs;
      values8(e[i], u[i]);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        acc[i][j] = fmaf(d[i][j], u[i][j], acc[i][j]);
        d[i][j] *= wt[j];
        dot = fmaf(d[i][j], u[i][j], dot);
      }
    }
    dot = row_sum<NT>(dot, sh[k & 1]) / (float)cols;
#pragma unroll
    for (int i = 0; i < kCh; ++i) {
#pragma unroll
      for (int j = 0; j < 8; ++j) d[i][j] = rs * fmaf(-u[i][j], dot, d[i][j]);
      const int n = left8(cols, column(i));
      if (n > 0) store8(static_cast<T*>(dx.p) + r * dx.ld, column(i), n, true, d[i]);
    }
  }
  if (part) {
    if constexpr (NT == 32) {  // the CTA's eight rows of sums to one, in order
      constexpr int kSpan = kCh * NT * 8;
      static_assert(RPC * kSpan * 4 <= kStage * (kAhead + 1), "the stages hold the rows of sums");
      float* joined = reinterpret_cast<float*>(stages);
      copies_wait<0>();
      __syncthreads();  // no stage is in use
#pragma unroll
      for (int i = 0; i < kCh; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) joined[threadIdx.x / NT * kSpan + column(i) + j] = acc[i][j];
      __syncthreads();
      for (int c = threadIdx.x; c < cols; c += THREADS) {
        float v = joined[c];
#pragma unroll
        for (int w8 = 1; w8 < RPC; ++w8) v += joined[w8 * kSpan + c];
        part[(int64_t)blockIdx.x * ld_part + c] = v;
      }
    } else {
#pragma unroll
      for (int i = 0; i < kCh; ++i)
        if (left8(cols, column(i)) > 0) store8(part + (int64_t)blockIdx.x * ld_part, column(i), 8, true, acc[i]);
    }
  }
}

// ---- rows too wide for a CTA's registers (more than 16384 columns): two passes over the row
constexpr int kWide = 512;

template <typename T>
__global__ void __launch_bounds__(kWide)
    rms_fwd_wide_kernel(Mat x, int64_t rows, int64_t cols, const void* __restrict__ w, bool w_f32, float eps, Mat y,
                        Saved S, float* rstd) {
  __shared__ float sh[2][kWide / 32];
  const int lane = threadIdx.x & (kLanes - 1);
  int k = 0;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x, ++k) {
    const T* row = static_cast<const T*>(x.p) + r * x.ld;
    float ss = 0.0f;
    for (int64_t c = threadIdx.x * 8; c < cols; c += kWide * 8) {
      float f[8];
      unpack8(load8(row, c, left8(cols, c)), f);
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = fmaf(f[j], f[j], ss);
    }
    ss = row_sum<kWide>(ss, sh[k & 1]);
    const float rs = rsqrtf(ss / (float)cols + eps);
    if (threadIdx.x == 0 && rstd) rstd[r] = rs;
    for (int64_t cc = 0; cc < cols; cc += kWide * 8) {  // every lane, for the shuffles
      const int64_t c = cc + threadIdx.x * 8, c0 = c - 8 * lane;
      const int n = left8(cols, c);
      float f[8], wt[8];
      const Oct<T> o = load8(row, c, n);
      unpack8(o, f);
      if (S.q) {
        const float amax[1] = {block_amax(o)};
        float gain[1];
        const float scale = block_gains(amax, gain);
        if (n > 0) __stcs(reinterpret_cast<uint2*>(S.q + r * S.ld_q + c), quant8(f, gain[0]));
        if (lane == 0 && c0 < cols) S.scale[r * S.ld_s + c0 / kBlock] = scale;
      }
      load_weight<T>(w, w_f32, cols, c, wt);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = f[j] * rs * wt[j];
      if (n > 0) store8(static_cast<T*>(y.p) + r * y.ld, c, n, true, f);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kWide)
    rms_bwd_wide_kernel(Mat dy, int64_t rows, int64_t cols, const void* __restrict__ w, bool w_f32, Saved S,
                        const float* __restrict__ rstd, Mat dx, float* part, int64_t ld_part) {
  __shared__ float sh[2][kWide / 32];
  float* mine = part ? part + blockIdx.x * ld_part : nullptr;
  int k = 0;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x, ++k) {
    const T* row = static_cast<const T*>(dy.p) + r * dy.ld;
    const float rs = rstd[r];
    float dot = 0.0f;
    for (int64_t c = threadIdx.x * 8; c < cols; c += kWide * 8) {
      const int n = left8(cols, c);
      float d[8], u[8], wt[8];
      unpack8(load8(row, c, n), d);
      Eights e = fetch8(S, r, c, n);
      e.s *= rs;
      values8(e, u);
      load_weight<T>(w, w_f32, cols, c, wt);
      if (mine) {  // a thread owns its columns of the CTA's sums: plain loads and stores, no atomics
        float4* at = reinterpret_cast<float4*>(mine + c);
        float4 s0 = make_float4(0.0f, 0.0f, 0.0f, 0.0f), s1 = s0;
        if (k) s0 = at[0], s1 = at[1];
        at[0] = make_float4(fmaf(d[0], u[0], s0.x), fmaf(d[1], u[1], s0.y), fmaf(d[2], u[2], s0.z), fmaf(d[3], u[3], s0.w));
        at[1] = make_float4(fmaf(d[4], u[4], s1.x), fmaf(d[5], u[5], s1.y), fmaf(d[6], u[6], s1.z), fmaf(d[7], u[7], s1.w));
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) dot = fmaf(d[j] * wt[j], u[j], dot);
    }
    dot = row_sum<kWide>(dot, sh[k & 1]) / (float)cols;
    for (int64_t c = threadIdx.x * 8; c < cols; c += kWide * 8) {
      const int n = left8(cols, c);
      float d[8], u[8], wt[8];
      unpack8(load8(row, c, n), d);
      Eights e = fetch8(S, r, c, n);
      e.s *= rs;
      values8(e, u);
      load_weight<T>(w, w_f32, cols, c, wt);
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
int bpr_log2_of(int64_t cols) {
  const int64_t blocks = (cols + kBlock - 1) / kBlock;
  int l = 0;
  while (l < 4 && (1 << l) < blocks) ++l;
  return l;
}
// As many CTAs as are resident (eight of 256 threads per SM), each walking down its rows.
dim3 block_grid(int64_t rows, int64_t cols, int bpr_log2, int unroll) {
  const int64_t blocks = (cols + kBlock - 1) / kBlock, rpc = (int64_t)(kHalves >> bpr_log2) * unroll;
  const int64_t gx = std::min<int64_t>((blocks + (1 << bpr_log2) - 1) >> bpr_log2, 65535);
  const int64_t most = std::max<int64_t>(1, (int64_t)eco_num_sms() * 8 / gx);
  const int64_t gy = std::min<int64_t>((rows + rpc - 1) / rpc, std::min<int64_t>(most, 65535));
  return dim3((unsigned)gx, (unsigned)gy);
}

int check_saved(const eco_saved_i8_t* S, int64_t rows, int64_t cols, const char* who) {
  ECO_REQUIRE(S && S->q && S->scale && S->ld_q >= cols && S->ld_q % 16 == 0 && eco_aligned16(S->q) &&
                  S->ld_scale >= (cols + kBlock - 1) / kBlock,
              ECO_ERR_ARG, "%s: bad eight-bit buffers", who);
  return ECO_OK;
}
Saved saved_of(const eco_saved_i8_t* S) {
  return S ? Saved{S->q, S->scale, S->ld_q, S->ld_scale} : Saved{nullptr, nullptr, 0, 0};
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
int check_in(const void* p, int64_t ld, int64_t rows, int64_t cols, int type, const char* who) {
  ECO_REQUIRE(p && (rows <= 1 || ld >= 0) && reinterpret_cast<uintptr_t>(p) % (uintptr_t)es_of(type) == 0, ECO_ERR_ARG,
              "%s: bad input", who);
  return ECO_OK;
}
// Outputs have rows of whole groups of eight columns that start on a boundary of their size.
int check_out(const void* p, int64_t ld, int64_t rows, int64_t cols, int type, const char* who) {
  ECO_REQUIRE(p && ld >= (cols + 7) / 8 * 8, ECO_ERR_ARG, "%s: output rows too short", who);
  ECO_REQUIRE(rows_on_8(p, ld, 2, type), ECO_ERR_MISALIGNED, "%s: output rows do not start on eight elements", who);
  return ECO_OK;
}
int check_shape(int64_t rows, int64_t cols, int type, const char* who) {
  ECO_REQUIRE(rows >= 0 && cols > 0 && cols <= (int64_t)1 << 28, ECO_ERR_ARG, "%s: bad shape", who);
  ECO_REQUIRE(good_type(type), ECO_ERR_ARG, "%s: unknown type %d", who, type);
  return ECO_OK;
}

template <typename F>
void by_float(int type, F f) {
  if (type == ECO_F32) f((float*)nullptr);
  else if (type == ECO_BF16) f((__nv_bfloat16*)nullptr);
  else f((__half*)nullptr);
}

// Threads of a row (16 columns each), 0 for the two-pass kernels of wider rows.
int row_threads(int64_t cols) {
  int nt = 32;
  while (nt < 1024 && (int64_t)nt * 8 * kCh < cols) nt *= 2;
  return (int64_t)nt * 8 * kCh < cols ? 0 : nt;
}
template <typename F>
void by_width(int64_t cols, F f) {
  switch (row_threads(cols)) {
    case 32: return f(std::integral_constant<int, 32>{});
    case 64: return f(std::integral_constant<int, 64>{});
    case 128: return f(std::integral_constant<int, 128>{});
    case 256: return f(std::integral_constant<int, 256>{});
    case 512: return f(std::integral_constant<int, 512>{});
    case 1024: return f(std::integral_constant<int, 1024>{});
    default: return f(std::integral_constant<int, 0>{});
  }
}
// CTAs of the norm's kernels: what is resident at 1024 threads per SM.
int64_t rms_ctas(int64_t rows, int64_t cols) {
  const int nt = row_threads(cols);
  const int threads = nt == 0 ? kWide : nt == 32 ? kThreads : nt, rpc = nt == 32 ? kThreads / 32 : 1;
  return std::min<int64_t>((rows + rpc - 1) / rpc, (int64_t)eco_num_sms() * (1024 / threads));
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
    pack_kernel<T, U><<<block_grid(rows, cols, l, U), kThreads, 0, eco_stream(stream)>>>(
        Mat{const_cast<void*>(x), ld}, rows, cols, saved_of(saved), l);
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
    restore_kernel<T, 4><<<block_grid(rows, cols, l, 4), kThreads, 0, eco_stream(stream)>>>(saved_of(saved), rows,
                                                                                            cols, Mat{x, ld}, l);
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
    const Mat g{const_cast<void*>(gate), ld_gate}, u{const_cast<void*>(up), ld_up}, o{y, ld_y};
    if (act == ECO_ACT_GELU)
      gated_fwd_kernel<T, true, U><<<grid, kThreads, 0, eco_stream(stream)>>>(g, u, rows, cols, o, saved_of(saved_gate),
                                                                           saved_of(saved_up), l);
    else
      gated_fwd_kernel<T, false, U><<<grid, kThreads, 0, eco_stream(stream)>>>(g, u, rows, cols, o, saved_of(saved_gate),
                                                                            saved_of(saved_up), l);
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
  ECO_REQUIRE(dgate && dup && (rows <= 1 || (ld_dgate >= cols && ld_dup >= cols)), ECO_ERR_ARG,
              "eco_gated_act_bwd: bad outputs");
  // A half of one packed output has no padding of its own: the last columns, fewer than eight,
  // are stored one by one, and so is a half whose rows do not start on eight elements.
  const bool vg = rows_on_8(dgate, ld_dgate, rows, type);
  const bool vu = rows_on_8(dup, ld_dup, rows, type);
  const int l = bpr_log2_of(cols);
  by_float(type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    constexpr int U = sizeof(T) == 4 ? 1 : 2;
    const dim3 grid = block_grid(rows, cols, l, U);
    const Mat d{const_cast<void*>(dy), ld_dy}, g{dgate, ld_dgate}, u{dup, ld_dup};
    if (act == ECO_ACT_GELU)
      gated_bwd_kernel<T, true, U><<<grid, kThreads, 0, eco_stream(stream)>>>(
          d, rows, cols, saved_of(saved_gate), saved_of(saved_up), g, u, vg, vu, l);
    else
      gated_bwd_kernel<T, false, U><<<grid, kThreads, 0, eco_stream(stream)>>>(
          d, rows, cols, saved_of(saved_gate), saved_of(saved_up), g, u, vg, vu, l);
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
    by_width(cols, [&](auto nt) {
      constexpr int NT = decltype(nt)::value;
      const unsigned grid = (unsigned)rms_ctas(rows, cols);
      const Mat xi{const_cast<void*>(x), ld}, yo{y, ld_y};
      const bool w_f32 = w_type == ECO_F32;
      if constexpr (NT == 0) {
        rms_fwd_wide_kernel<T><<<grid, kWide, 0, eco_stream(stream)>>>(xi, rows, cols, w, w_f32, (float)eps, yo,
                                                                       saved_of(saved), rstd);
      } else {
        constexpr int threads = NT == 32 ? kThreads : NT, smem = Stage<T, false>::kBytes * threads * (Stage<T, false>::kAhead + 1);
        const bool async = rows_on_16(x, ld, rows, type);
        ok = allow_smem(rms_fwd_kernel<T, NT>, smem);
        if (ok)
          rms_fwd_kernel<T, NT><<<grid, threads, async ? smem : 0, eco_stream(stream)>>>(
              xi, rows, cols, w, w_f32, (float)eps, yo, saved_of(saved), rstd, async);
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
  ECO_REQUIRE(rstd, ECO_ERR_ARG, "eco_rms_norm_bwd: null rstd");
  const int64_t ctas = rms_ctas(rows, cols), ld_part = (cols + 7) / 8 * 8;
  ECO_REQUIRE(!dw || (scratch && eco_aligned16(scratch) && scratch_len >= ctas * ld_part), ECO_ERR_ARG,
              "eco_rms_norm_bwd: scratch too small (eco_rms_norm_bwd_scratch)");
  bool ok = true;
  by_float(type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    by_width(cols, [&](auto nt) {
      constexpr int NT = decltype(nt)::value;
      const unsigned grid = (unsigned)ctas;
      const Mat d{const_cast<void*>(dy), ld_dy}, o{dx, ld_dx};
      float* part = dw ? scratch : nullptr;
      const bool w_f32 = w_type == ECO_F32;
      if constexpr (NT == 0) {
        rms_bwd_wide_kernel<T><<<grid, kWide, 0, s>>>(d, rows, cols, w, w_f32, saved_of(saved), rstd, o, part, ld_part);
      } else {
        constexpr int threads = NT == 32 ? kThreads : NT, smem = Stage<T, true>::kBytes * threads * (Stage<T, true>::kAhead + 1);
        const bool async = rows_on_16(dy, ld_dy, rows, type);
        ok = allow_smem(rms_bwd_kernel<T, NT>, smem);
        if (ok)
          rms_bwd_kernel<T, NT><<<grid, threads, async || NT == 32 ? smem : 0, s>>>(d, rows, cols, w, w_f32, saved_of(saved), rstd,
                                                                        o, part, ld_part, async);
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
