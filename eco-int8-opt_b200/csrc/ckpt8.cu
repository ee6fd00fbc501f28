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
// on 16 bytes is read by the 16-byte words that hold its eight columns, shifted into place
// (each of them holds at least one of the eight, so none lies outside the row's memory).
template <typename T>
ECO_DEV Oct<T> load8(const T* row, int64_t c, int n) {
  constexpr int V = Oct<T>::W / 4;  // 16-byte words
  Oct<T> o;
  if (n == 8) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(row + c);
    const uint4* p = reinterpret_cast<const uint4*>(a & ~uintptr_t(15));
    const uint32_t skew = (uint32_t)a & 15;
    if (skew == 0) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const uint4 t = __ldg(p + v);
        o.w[4 * v] = t.x, o.w[4 * v + 1] = t.y, o.w[4 * v + 2] = t.z, o.w[4 * v + 3] = t.w;
      }
      return o;
    }
    uint32_t w[4 * V + 4];
#pragma unroll
    for (int v = 0; v <= V; ++v) {
      const uint4 t = __ldg(p + v);
      w[4 * v] = t.x, w[4 * v + 1] = t.y, w[4 * v + 2] = t.z, w[4 * v + 3] = t.w;
    }
    if (skew & 8) {
#pragma unroll
      for (int i = 0; i < 4 * V + 2; ++i) w[i] = w[i + 2];
    }
    if (skew & 4) {
#pragma unroll
      for (int i = 0; i < 4 * V + 1; ++i) w[i] = w[i + 1];
    }
    const uint32_t bits = (skew & 3) * 8;
#pragma unroll
    for (int i = 0; i < 4 * V; ++i) o.w[i] = __funnelshift_r(w[i], w[i + 1], bits);
    return o;
  }
#pragma unroll
  for (int i = 0; i < Oct<T>::W; ++i) o.w[i] = 0u;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n) {
      if constexpr (sizeof(T) == 4)
        o.w[i] = __float_as_uint(row[c + i]);
      else
        o.w[i / 2] |= (uint32_t)__ldg(reinterpret_cast<const unsigned short*>(row + c + i)) << (16 * (i & 1));
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

// Eight columns of an output row: whole vectors where the row starts on 16 bytes (its
// padding takes the rest of a last vector), else n single stores.
template <typename T>
ECO_DEV void store8(T* row, int64_t c, int n, bool vec, const float (&f)[8]) {
  if (vec) {
    uint4* p = reinterpret_cast<uint4*>(row + c);
    if constexpr (sizeof(T) == 4) {
      const float a[4] = {f[0], f[1], f[2], f[3]}, b[4] = {f[4], f[5], f[6], f[7]};
      p[0] = RowIo<T>::pack(a);
      if (n > 4) p[1] = RowIo<T>::pack(b);
    } else {
      p[0] = RowIo<T>::pack(f);
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
// max |x| of a block over its 16 lanes.
ECO_DEV float block_amax(const float (&f)[8]) {
  float m = fabsf(f[0]);
#pragma unroll
  for (int i = 1; i < 8; ++i) m = max_nan(m, fabsf(f[i]));
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  return m;
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
// Puts eight columns of a block away; all 16 lanes of the block call it.
ECO_DEV void put8(const float (&f)[8], int n, int8_t* q, int64_t c, float* scale) {
  const float amax = block_amax(f);
  const bool zero = amax < 0x1p-119f;  // false for NaN
  const float gain = zero ? 0.0f : __fdiv_rn(127.0f, amax);
  if (n > 0) __stcs(reinterpret_cast<uint2*>(q + c), quant8(f, gain));
  if ((threadIdx.x & (kLanes - 1)) == 0 && n > 0)
    *scale = zero ? 0.0f : (amax < INFINITY ? __fdiv_rn(amax, 127.0f) : __int_as_float(0x7fc00000));
}
ECO_DEV void get8(const int8_t* q, int64_t c, int n, const float* scale, float (&f)[8]) {
  uint2 w = make_uint2(0u, 0u);
  float s = 0.0f;
  if (n > 0) {
    w = __ldcs(reinterpret_cast<const uint2*>(q + c));
    s = __ldg(scale);
  }
  dequant8(w, f);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] *= s;
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
// Loops over (row, block) so that both halves of a warp stay in step (the shuffles need all
// 32 lanes): `body(row, block, first column, columns of this lane)`, no columns past the end.
template <typename F>
ECO_DEV void for_blocks(int64_t rows, int64_t cols, int bpr_log2, F body) {
  const Tile t(cols, bpr_log2);
  const int64_t first = (int64_t)blockIdx.y * (kHalves >> bpr_log2), firstb = (int64_t)blockIdx.x << bpr_log2;
  for (int64_t r = t.row0, rr = first; rr < rows; r += t.row_step, rr += t.row_step)
    for (int64_t b = t.b0, bb = firstb; bb < t.blocks; b += t.b_step, bb += t.b_step) {
      const int64_t c = b * kBlock + t.lane * 8;
      const int n = r < rows && b < t.blocks ? left8(cols, c) : 0;
      body(r, b, c, n);
    }
}

// ------------------------------------------------ put away, bring back
template <typename T>
__global__ void __launch_bounds__(kThreads) pack_kernel(Mat x, int64_t rows, int64_t cols, Saved S, int bpr_log2) {
  for_blocks(rows, cols, bpr_log2, [&](int64_t r, int64_t b, int64_t c, int n) {
    float f[8];
    unpack8(load8(static_cast<const T*>(x.p) + (n ? r * x.ld : 0), c, n), f);
    put8(f, n, S.q + r * S.ld_q, c, S.scale + r * S.ld_s + b);
  });
}

template <typename T>
__global__ void __launch_bounds__(kThreads) restore_kernel(Saved S, int64_t rows, int64_t cols, Mat x, int bpr_log2) {
  for_blocks(rows, cols, bpr_log2, [&](int64_t r, int64_t b, int64_t c, int n) {
    float f[8];
    get8(S.q + r * S.ld_q, c, n, S.scale + r * S.ld_s + b, f);
    if (n > 0) store8(static_cast<T*>(x.p) + r * x.ld, c, n, true, f);
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

template <typename T, bool GELU>
__global__ void __launch_bounds__(kThreads)
    gated_fwd_kernel(Mat gate, Mat up, int64_t rows, int64_t cols, Mat y, Saved SG, Saved SU, int bpr_log2) {
  for_blocks(rows, cols, bpr_log2, [&](int64_t r, int64_t b, int64_t c, int n) {
    const int64_t rr = n ? r : 0;
    const Oct<T> go = load8(static_cast<const T*>(gate.p) + rr * gate.ld, c, n);
    const Oct<T> uo = load8(static_cast<const T*>(up.p) + rr * up.ld, c, n);
    float g[8], u[8];
    unpack8(go, g);
    unpack8(uo, u);
    if (SG.q) {
      put8(g, n, SG.q + r * SG.ld_q, c, SG.scale + r * SG.ld_s + b);
      put8(u, n, SU.q + r * SU.ld_q, c, SU.scale + r * SU.ld_s + b);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) g[i] = g[i] * act_over_input<GELU>(g[i]) * u[i];
    if (n > 0) store8(static_cast<T*>(y.p) + r * y.ld, c, n, true, g);
  });
}

template <typename T, bool GELU>
__global__ void __launch_bounds__(kThreads)
    gated_bwd_kernel(Mat dy, int64_t rows, int64_t cols, Saved SG, Saved SU, Mat dgate, Mat dup, bool vec_g,
                     bool vec_u, int bpr_log2) {
  for_blocks(rows, cols, bpr_log2, [&](int64_t r, int64_t b, int64_t c, int n) {
    const Oct<T> d8 = load8(static_cast<const T*>(dy.p) + (n ? r * dy.ld : 0), c, n);
    float g[8], u[8], d[8];
    get8(SG.q + r * SG.ld_q, c, n, SG.scale + r * SG.ld_s + b, g);
    get8(SU.q + r * SU.ld_q, c, n, SU.scale + r * SU.ld_s + b, u);
    unpack8(d8, d);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float s = act_over_input<GELU>(g[i]);
      const float dg = d[i] * u[i] * act_slope<GELU>(g[i], s);
      u[i] = d[i] * g[i] * s;
      g[i] = dg;
    }
    if (n > 0) {
      store8(static_cast<T*>(dgate.p) + r * dgate.ld, c, n, vec_g && n == 8, g);
      store8(static_cast<T*>(dup.p) + r * dup.ld, c, n, vec_u && n == 8, u);
    }
  });
}

// ------------------------------------------------ rms norm
// y = x r w,  r = 1 / sqrt(mean x^2 + eps);  with x' = what the eight bits stand for, u = x' r:
//   dx = r (w dy - u mean(w dy u)),   dw = sum over rows of dy u.
//
// NT threads hold a row (CH groups of eight columns each), so a row is read once; the sum is
// joined over the threads in a fixed order.  Rows wider than that (CH == 0) are read again
// for the second pass, and their dw sums live in the CTA's own row of `part`.
template <int NT>
ECO_DEV float row_sum(float v, float* sh) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (NT > 32) {
    constexpr int W = NT / 32;
    __syncthreads();  // sh may still be read for the row before
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    v = sh[threadIdx.x % W];
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  }
  return v;
}

template <typename T, typename WT, int NT, int CH>
__global__ void __launch_bounds__(NT == 32 ? kThreads : NT)
    rms_fwd_kernel(Mat x, int64_t rows, int64_t cols, const WT* __restrict__ w, float eps, Mat y, Saved S,
                   float* rstd) {
  __shared__ float sh[NT / 32];
  constexpr int RPC = NT == 32 ? kThreads / NT : 1;  // a wider row has the CTA's barriers to itself
  const int tid = threadIdx.x % NT;
  const int64_t span = (int64_t)NT * 8;
  const int chunks = CH > 0 ? CH : (int)((cols + span - 1) / span);
  for (int64_t r = (int64_t)blockIdx.x * RPC + threadIdx.x / NT; r < rows; r += (int64_t)gridDim.x * RPC) {
    const T* row = static_cast<const T*>(x.p) + r * x.ld;
    Oct<T> keep[CH > 0 ? CH : 1];
    if constexpr (CH > 0) {
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const int64_t c = i * span + tid * 8;
        keep[i] = load8(row, c, left8(cols, c));
      }
    }
    float ss = 0.0f;
#pragma unroll(CH > 0 ? CH : 1)
    for (int i = 0; i < chunks; ++i) {
      const int64_t c = i * span + tid * 8;
      float f[8];
      unpack8(CH > 0 ? keep[CH > 0 ? i : 0] : load8(row, c, left8(cols, c)), f);
#pragma unroll
      for (int k = 0; k < 8; ++k) ss = fmaf(f[k], f[k], ss);
    }
    ss = row_sum<NT>(ss, sh);
    const float rs = rsqrtf(ss / (float)cols + eps);
    if (tid == 0 && rstd) rstd[r] = rs;
#pragma unroll(CH > 0 ? CH : 1)
    for (int i = 0; i < chunks; ++i) {
      const int64_t c = i * span + tid * 8;
      const int n = left8(cols, c);
      float f[8], g[8];
      unpack8(CH > 0 ? keep[CH > 0 ? i : 0] : load8(row, c, n), f);
      if (S.q) put8(f, n, S.q + r * S.ld_q, c, S.scale + r * S.ld_s + c / kBlock);
      if (w) unpack8(load8(w, c, n), g);
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] = w ? f[k] * rs * g[k] : f[k] * rs;
      if (n > 0) store8(static_cast<T*>(y.p) + r * y.ld, c, n, true, f);
    }
  }
}

template <typename T, typename WT, int NT, int CH>
__global__ void __launch_bounds__(NT == 32 ? kThreads : NT)
    rms_bwd_kernel(Mat dy, int64_t rows, int64_t cols, const WT* __restrict__ w, Saved S,
                   const float* __restrict__ rstd, Mat dx, float* part, int64_t ld_part) {
  __shared__ float sh[NT / 32];
  constexpr int RPC = NT == 32 ? kThreads / NT : 1;  // a wider row has the CTA's barriers to itself
  const int tid = threadIdx.x % NT;
  const int64_t span = (int64_t)NT * 8;
  const int chunks = CH > 0 ? CH : (int)((cols + span - 1) / span);
  float acc[CH > 0 ? CH : 1][8] = {};
  // one row of `part` per row group of the grid
  float* mine = part ? part + ((int64_t)blockIdx.x * RPC + threadIdx.x / NT) * ld_part : nullptr;
  if (CH == 0 && mine)
    for (int i = 0; i < chunks; ++i) {
      const int64_t c = i * span + tid * 8;
      if (left8(cols, c) > 0) store8(mine, c, 8, true, acc[0]);
    }
  for (int64_t r = (int64_t)blockIdx.x * RPC + threadIdx.x / NT; r < rows; r += (int64_t)gridDim.x * RPC) {
    const T* drow = static_cast<const T*>(dy.p) + r * dy.ld;
    const int8_t* qrow = S.q + r * S.ld_q;
    const float* srow = S.scale + r * S.ld_s;
    const float rs = rstd[r];
    Oct<T> keep[CH > 0 ? CH : 1];
    uint2 bytes[CH > 0 ? CH : 1];
    float unit[CH > 0 ? CH : 1];  // scale * rstd
    auto fetch = [&](int64_t c, Oct<T>& o, uint2& q, float& s) {
      const int n = left8(cols, c);
      o = load8(drow, c, n);
      q = make_uint2(0u, 0u);
      s = 0.0f;
      if (n > 0) {
        q = __ldcs(reinterpret_cast<const uint2*>(qrow + c));
        s = __ldg(srow + c / kBlock) * rs;
      }
    };
    if constexpr (CH > 0) {
#pragma unroll
      for (int i = 0; i < CH; ++i) fetch(i * span + tid * 8, keep[i], bytes[i], unit[i]);
    }
    float dot = 0.0f;
#pragma unroll(CH > 0 ? CH : 1)
    for (int i = 0; i < chunks; ++i) {
      const int64_t c = i * span + tid * 8;
      const int j = CH > 0 ? i : 0;
      if (CH == 0) fetch(c, keep[0], bytes[0], unit[0]);
      float d[8], u[8], g[8];
      unpack8(keep[j], d);
      dequant8(bytes[j], u);
      if (w) unpack8(load8(w, c, left8(cols, c)), g);
      if (CH == 0 && mine && left8(cols, c) > 0) {  // plain loads: the CTA writes this row itself
#pragma unroll
        for (int k = 0; k < 8; ++k) acc[0][k] = mine[c + k];
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        u[k] *= unit[j];
        acc[j][k] = fmaf(d[k], u[k], acc[j][k]);
        dot = fmaf(w ? d[k] * g[k] : d[k], u[k], dot);
      }
      if (CH == 0 && mine && left8(cols, c) > 0) store8(mine, c, 8, true, acc[0]);
    }
    dot = row_sum<NT>(dot, sh) / (float)cols;
#pragma unroll(CH > 0 ? CH : 1)
    for (int i = 0; i < chunks; ++i) {
      const int64_t c = i * span + tid * 8;
      const int n = left8(cols, c), j = CH > 0 ? i : 0;
      if (CH == 0) fetch(c, keep[0], bytes[0], unit[0]);
      float d[8], u[8], g[8];
      unpack8(keep[j], d);
      dequant8(bytes[j], u);
      if (w) unpack8(load8(w, c, n), g);
#pragma unroll
      for (int k = 0; k < 8; ++k) d[k] = rs * fmaf(-u[k] * unit[j], dot, w ? d[k] * g[k] : d[k]);
      if (n > 0) store8(static_cast<T*>(dx.p) + r * dx.ld, c, n, true, d);
    }
  }
  if (CH > 0 && mine) {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int64_t c = i * span + tid * 8;
      if (left8(cols, c) > 0) store8(mine, c, 8, true, acc[i]);
    }
  }
}

// dw = column sums of the `n` partial rows, in double and in order: 32 columns x 8 rows of
// threads per CTA.
template <typename WT>
__global__ void __launch_bounds__(256) rms_dw_kernel(const float* __restrict__ part, int64_t n, int64_t ld_part,
                                                      int64_t cols, WT* dw) {
  __shared__ double sh[8][33];
  const int lane = threadIdx.x & 31, q = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane;
  double v = 0.0;
  if (c < cols)
    for (int64_t i = q; i < n; i += 8) v += part[i * ld_part + c];
  sh[q][lane] = v;
  __syncthreads();
  if (q == 0 && c < cols) {
    for (int i = 1; i < 8; ++i) v += sh[i][lane];
    dw[c] = from_f32<WT>((float)v);
  }
}

// ------------------------------------------------ host side
int bpr_log2_of(int64_t cols) {
  const int64_t blocks = (cols + kBlock - 1) / kBlock;
  int l = 0;
  while (l < 4 && (1 << l) < blocks) ++l;
  return l;
}
dim3 block_grid(int64_t rows, int64_t cols, int bpr_log2) {
  const int64_t blocks = (cols + kBlock - 1) / kBlock, rpc = kHalves >> bpr_log2;
  const int64_t gx = std::min<int64_t>((blocks + (1 << bpr_log2) - 1) >> bpr_log2, 65535);
  const int64_t gy = std::min<int64_t>((rows + rpc - 1) / rpc, 65535);
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
int check_in(const void* p, int64_t ld, int64_t rows, int64_t cols, int type, const char* who) {
  ECO_REQUIRE(p && (rows <= 1 || ld >= 0) && reinterpret_cast<uintptr_t>(p) % (uintptr_t)es_of(type) == 0, ECO_ERR_ARG,
              "%s: bad input", who);
  return ECO_OK;
}
// Outputs have rows that start on 16 bytes and room for whole vectors behind the last column.
int check_out(const void* p, int64_t ld, int64_t rows, int64_t cols, int type, const char* who) {
  const int64_t per = 16 / es_of(type);
  ECO_REQUIRE(p && ld >= (cols + per - 1) / per * per, ECO_ERR_ARG, "%s: output rows too short", who);
  ECO_REQUIRE(rows_on_16(p, ld, 2, type), ECO_ERR_MISALIGNED, "%s: output rows do not start on 16 bytes", who);
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

// Threads and groups of a row: four groups of eight columns per thread as far as a CTA goes.
template <typename F>
void by_width(int64_t cols, F f) {
  if (cols <= 256) f(std::integral_constant<int, 32>{}, std::integral_constant<int, 1>{});
  else if (cols <= 1024) f(std::integral_constant<int, 128>{}, std::integral_constant<int, 1>{});
  else if (cols <= 4096) f(std::integral_constant<int, 128>{}, std::integral_constant<int, 4>{});
  else if (cols <= 8192) f(std::integral_constant<int, 256>{}, std::integral_constant<int, 4>{});
  else if (cols <= 16384) f(std::integral_constant<int, 512>{}, std::integral_constant<int, 4>{});
  else f(std::integral_constant<int, 512>{}, std::integral_constant<int, 0>{});
}
int row_threads(int64_t cols) { return cols <= 256 ? 32 : cols <= 4096 ? 128 : cols <= 8192 ? 256 : 512; }
int64_t rms_groups(int64_t rows, int64_t cols) {  // row groups of the backward's grid
  const int nt = row_threads(cols), threads = nt == 32 ? kThreads : nt, rpc = threads / nt;
  const int64_t ctas = std::min<int64_t>((rows + rpc - 1) / rpc, (int64_t)eco_num_sms() * (1024 / threads));
  return ctas * rpc;
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
    pack_kernel<T><<<block_grid(rows, cols, l), kThreads, 0, eco_stream(stream)>>>(
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
    restore_kernel<T><<<block_grid(rows, cols, l), kThreads, 0, eco_stream(stream)>>>(saved_of(saved), rows, cols,
                                                                                      Mat{x, ld}, l);
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
  const dim3 grid = block_grid(rows, cols, l);
  by_float(type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    const Mat g{const_cast<void*>(gate), ld_gate}, u{const_cast<void*>(up), ld_up}, o{y, ld_y};
    if (act == ECO_ACT_GELU)
      gated_fwd_kernel<T, true><<<grid, kThreads, 0, eco_stream(stream)>>>(g, u, rows, cols, o, saved_of(saved_gate),
                                                                           saved_of(saved_up), l);
    else
      gated_fwd_kernel<T, false><<<grid, kThreads, 0, eco_stream(stream)>>>(g, u, rows, cols, o, saved_of(saved_gate),
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
  // are stored one by one, and so is a half whose rows do not start on 16 bytes.
  const bool vg = rows_on_16(dgate, ld_dgate, rows, type);
  const bool vu = rows_on_16(dup, ld_dup, rows, type);
  const int l = bpr_log2_of(cols);
  const dim3 grid = block_grid(rows, cols, l);
  by_float(type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    const Mat d{const_cast<void*>(dy), ld_dy}, g{dgate, ld_dgate}, u{dup, ld_dup};
    if (act == ECO_ACT_GELU)
      gated_bwd_kernel<T, true><<<grid, kThreads, 0, eco_stream(stream)>>>(
          d, rows, cols, saved_of(saved_gate), saved_of(saved_up), g, u, vg, vu, l);
    else
      gated_bwd_kernel<T, false><<<grid, kThreads, 0, eco_stream(stream)>>>(
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
  by_float(type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    by_width(cols, [&](auto nt, auto ch) {
      constexpr int NT = decltype(nt)::value, CH = decltype(ch)::value;
      constexpr int threads = NT == 32 ? kThreads : NT, rpc = threads / NT;
      const unsigned grid = (unsigned)std::min<int64_t>((rows + rpc - 1) / rpc, (int64_t)eco_num_sms() * 8);
      const Mat xi{const_cast<void*>(x), ld}, yo{y, ld_y};
      if (w && w_type != type)
        rms_fwd_kernel<T, float, NT, CH><<<grid, threads, 0, eco_stream(stream)>>>(
            xi, rows, cols, static_cast<const float*>(w), (float)eps, yo, saved_of(saved), rstd);
      else
        rms_fwd_kernel<T, T, NT, CH><<<grid, threads, 0, eco_stream(stream)>>>(
            xi, rows, cols, static_cast<const T*>(w), (float)eps, yo, saved_of(saved), rstd);
    });
  });
  return eco_launch_check("eco_rms_norm");
}

extern "C" int64_t eco_rms_norm_bwd_scratch(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0) return 0;
  return rms_groups(rows, cols) * ((cols + 7) / 8 * 8);
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
  const int64_t groups = rms_groups(rows, cols), ld_part = (cols + 7) / 8 * 8;
  ECO_REQUIRE(!dw || (scratch && eco_aligned16(scratch) && scratch_len >= groups * ld_part), ECO_ERR_ARG,
              "eco_rms_norm_bwd: scratch too small (eco_rms_norm_bwd_scratch)");
  by_float(type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    by_width(cols, [&](auto nt, auto ch) {
      constexpr int NT = decltype(nt)::value, CH = decltype(ch)::value;
      constexpr int threads = NT == 32 ? kThreads : NT, rpc = threads / NT;
      const unsigned grid = (unsigned)(groups / rpc);
      const Mat d{const_cast<void*>(dy), ld_dy}, o{dx, ld_dx};
      float* part = dw ? scratch : nullptr;
      if (w && w_type != type)
        rms_bwd_kernel<T, float, NT, CH><<<grid, threads, 0, s>>>(d, rows, cols, static_cast<const float*>(w),
                                                                  saved_of(saved), rstd, o, part, ld_part);
      else
        rms_bwd_kernel<T, T, NT, CH><<<grid, threads, 0, s>>>(d, rows, cols, static_cast<const T*>(w),
                                                              saved_of(saved), rstd, o, part, ld_part);
    });
  });
  if (dw)
    by_float(w_type, [&](auto* t) {
      using WT = std::remove_pointer_t<decltype(t)>;
      rms_dw_kernel<WT><<<(unsigned)((cols + 31) / 32), 256, 0, s>>>(scratch, groups, ld_part, cols,
                                                                     static_cast<WT*>(dw));
    });
  return eco_launch_check("eco_rms_norm_bwd");
}
