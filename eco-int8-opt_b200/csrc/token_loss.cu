// Objectives on the log-probabilities of given tokens, from logits, with their gradient:
// the token log-probabilities themselves, a clipped policy loss with a KL term, and a loss
// over pairs of log ratios.
//
// For a row x of `cols` logits (x = raw * mul: the temperature, and the scale of int8
// logits) and its token y:
//
//   lp = x_y - log sum_j exp x_j;          d lp / d x_j = [j = y] - p_j,  p = softmax(x)
//
// so the gradient of any objective L(lp_0, lp_1, ...) is one coefficient per row,
// c_r = dL/dlp_r, times ([j = y] - p_j).  Rows that do not count (masked, or a token outside
// [0, cols)) are never read: their logits may hold anything; their gradient rows are zeros.
//
// A row is one online pass (running max m and s = sum 2^((x - m) log2 e), rescaled when m
// grows) and, for the gradient, one pass that writes -c/s 2^((x - m) log2 e) (+ c at y).
// Sums are fp32 per thread over its share of the row and joined in a fixed order; the log of
// the sum and the token's term meet in double, once per row, because exp(ref - lp) - (ref - lp)
// - 1 loses what fp32 loses twice over.
#include <algorithm>
#include <cmath>

#include "abi.cuh"
#include "common.cuh"
#include "rowio.cuh"

namespace {

ECO_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// exp((x - m) mul) = 2^((x - m) c), c = mul log2 e.  The sum takes c in two parts: rounded to
// one, it would stretch every difference by the same 2^-26 or so, which 10^5 terms do not
// average out; the gradient's single probabilities do with one.
struct Factor {
  float hi, lo;
};
// What is subtracted before the exponential: m, and 0 for -inf alone (whose terms are then 0).
// x - m comes first and is multiplied after: a row masked to its type's lowest value would
// leave the fp32 range as x * c, and as x - m is 0 or -inf.
ECO_DEV float row_off(float m) { return m == -INFINITY ? 0.0f : m; }
ECO_DEV float term(float x, float off, Factor c) {
  const float d = x - off;
  return ex2(fmaf(d, c.lo, d * c.hi));
}

struct MaxSum {
  float m, s;
};
// Joined over W lanes (a power of two; groups side by side); every lane gets the same bits.
template <int W>
ECO_DEV MaxSum lanes_join(MaxSum a, Factor c) {
  float m = a.m;
  if (W == 32) {
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(a.m));
  } else {
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  }
  float s = a.s * term(a.m, row_off(m), c);
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return MaxSum{m, s};
}

template <int E>
ECO_DEV void take(MaxSum& a, const float (&x)[E], Factor c) {
  float vm = x[0];
#pragma unroll
  for (int k = 1; k < E; ++k) vm = fmaxf(vm, x[k]);
  if (vm > a.m) {
    a.s *= term(a.m, vm, c);
    a.m = vm;
  }
  const float off = row_off(a.m);
#pragma unroll
  for (int k = 0; k < E; ++k) a.s += term(x[k], off, c);
}
// What a row's gradient needs: g_j = -k 2^((x_j - off) c), and coef more at the token.
struct Slope {
  float off, c, k, coef;
  float base;  // 16-bit gradients: log2 |k| - off c, or NaN where that would cost accuracy
};
ECO_DEV Slope slope_of(float off, float c, float k, float coef) {
  const float t = off * c;
  return Slope{off, c, k, coef, fabsf(t) < 512.0f ? log2f(fabsf(k)) - t : __int_as_float(0x7fc00000)};
}
// A vector's logits to the vector of their gradient (without the token's share), stored at g + v E.
// FOLD, 16 bits: |k| goes into the exponent, so that an element costs one multiply-add, one
// exponential and half of a pack and a sign flip.  Its rounding is |exponent| 2^-24 and with
// |off c| < 512 at most 2^-15 of the value, against half a step of 2^-9 or 2^-11.
template <typename T, bool FOLD>
ECO_DEV void store_slope(typename RowIo<T>::G* g, int64_t v, const uint4& raw, const Slope& w) {
  constexpr int E = RowIo<T>::E;
  float f[E];
  RowIo<T>::unpack(raw, f);
  if constexpr (FOLD && sizeof(T) == 2) {
    if (w.base == w.base) {  // the same for the whole row
#pragma unroll
      for (int i = 0; i < E; ++i) f[i] = ex2(fmaf(f[i], w.c, w.base));
      uint4 q = RowIo<T>::pack(f);
      const uint32_t sign = w.k > 0.0f ? 0x80008000u : 0u;
      q.x ^= sign, q.y ^= sign, q.z ^= sign, q.w ^= sign;
      __stcs(reinterpret_cast<uint4*>(g) + v, q);
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < E; ++i) f[i] = -w.k * ex2((f[i] - w.off) * w.c);
  RowIo<T>::store(g, v, f);
}
// One element of it, the token's share included.
ECO_DEV float slope_at(float x, const Slope& w, bool token) {
  const float e = ex2((x - w.off) * w.c);
  return token ? fmaf(-w.k, e, w.coef) : -w.k * e;
}

// N vectors at a time: their maximum first, so that the terms depend on nothing but it (and the
// sum is rescaled only where the maximum has grown: seldom, after the first few).  ALL: all of
// them count; else `in` says which, and the others are worked on for nothing (lanes of a warp
// differ in it: a branch would run both ways).
template <typename T, bool ALL, int N>
ECO_DEV void take_vectors(MaxSum& a, const uint4 (&raw)[N], const bool (&in)[N], Factor c) {
  constexpr int E = RowIo<T>::E;
  float m = a.m;
#pragma unroll
  for (int p = 0; p < N; ++p) m = ALL || in[p] ? fmaxf(m, RowIo<T>::max(raw[p])) : m;
  const float off = row_off(m);
  if (m > a.m) {
    a.s *= term(a.m, off, c);
    a.m = m;
  }
#pragma unroll
  for (int p = 0; p < N; ++p) {
    float f[E], s[2] = {0.0f, 0.0f};
    RowIo<T>::unpack(raw[p], f);
#pragma unroll
    for (int k = 0; k < E; ++k) s[k & 1] += term(f[k], off, c);
    a.s += ALL || in[p] ? s[0] + s[1] : 0.0f;
  }
}
// Vectors p, p + step, ... of which `left` (counted in steps, from p on) count; N at a time.
template <typename T, int N, bool SHARED>
ECO_DEV void take_run(MaxSum& a, const uint4* p, int step, int left, Factor c) {
  uint4 raw[N];
  bool in[N];
  for (; left >= N; left -= N, p += N * step) {
#pragma unroll
    for (int u = 0; u < N; ++u) raw[u] = SHARED ? p[u * step] : __ldg(p + u * step);
    take_vectors<T, true, N>(a, raw, in, c);
  }
  if (left > 0) {
#pragma unroll
    for (int u = 0; u < N; ++u) {
      in[u] = u < left;
      raw[u] = in[u] ? (SHARED ? p[u * step] : __ldg(p + u * step)) : make_uint4(0u, 0u, 0u, 0u);
    }
    take_vectors<T, false, N>(a, raw, in, c);
  }
}
// How many of the vectors tid, tid + NT, ... lie below `vecs`.
template <int NT>
ECO_DEV int run_length(int vecs, int tid) { return vecs > tid ? (vecs - tid + NT - 1) / NT : 0; }

template <typename T, int NT>
ECO_DEV void row_grad(const T* x, typename RowIo<T>::G* g, int64_t cols, const Slope& w, int64_t y, int64_t tid,
                      int64_t v_end) {
  constexpr int E = RowIo<T>::E;
  using G = typename RowIo<T>::G;
  const RowSplit sp = RowIo<T>::split(x, cols);
  const T* body = x + sp.head;
  G* gb = g + sp.head;
  const int vend = (int)(v_end < sp.vecs ? v_end : sp.vecs);
  for (int v0 = (int)tid; v0 < vend; v0 += 4 * NT) {
    uint4 r[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (v0 + u * NT < vend) r[u] = RowIo<T>::load_last(body, v0 + u * NT);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int v = v0 + u * NT;
      if (v >= vend) break;
      store_slope<T, false>(gb, v, r[u], w);
      const int d = (int)y - sp.head - v * E;
      // the token's element, by the thread that has just written its vector
      if (d >= 0 && d < E) gb[v * E + d] = from_f32<G>(slope_at(to_f32(body[v * E + d]), w, true));
    }
  }
  if (tid < sp.head + sp.tail) {  // the threads of the row's first segment
    const int64_t j = sp.edge((int)tid, cols);
    g[j] = from_f32<G>(slope_at(to_f32(x[j]), w, j == y));
  }
}

template <typename T, int NT>
ECO_DEV void row_zero(const T* x, typename RowIo<T>::G* g, int64_t cols, int64_t tid, int64_t v_end) {
  constexpr int E = RowIo<T>::E;
  const RowSplit sp = RowIo<T>::split(x, cols);
  const int64_t vend = v_end < sp.vecs ? v_end : sp.vecs;
  const float f[E] = {};
  for (int64_t v = tid; v < vend; v += NT) RowIo<T>::store(g + sp.head, v, f);
  if (tid < sp.head + sp.tail) g[sp.edge((int)tid, cols)] = from_f32<typename RowIo<T>::G>(0.0f);
}

struct Rows {
  const void* x;
  int64_t rows, n1, s0, s1, cols;
  double mul;
  Factor c;  // mul * log2 e
  const int64_t* tokens;
  const uint8_t* mask;  // nullable
  const int32_t* cu;    // nullable: rows outside [cu[0], cu[nseq]) do not count
  int nseq;

  ECO_DEV int64_t at(int64_t r, int64_t t0, int64_t t1) const {
    if (n1 == rows) return r * t1;
    const int64_t o = r / n1;
    return o * t0 + (r - o * n1) * t1;
  }
  ECO_DEV bool counts(int64_t r) const {
    if (mask && !mask[r]) return false;
    const int64_t y = tokens[r];
    return y >= 0 && y < cols && (!cu || (r >= cu[0] && r < cu[nseq]));
  }
};
struct Grad {
  void* g;
  int64_t s0, s1;
};

// The row's term in double: (raw_y - m) mul - log s.  ex2 gives values that are 5.0e-8 of
// themselves too small on average (measured over arguments from -1 to -32, where it varies by
// 0.1e-8; 2^0 is exact).  A thread's own terms come out right on average, but every part of the
// sum that a join takes to a larger maximum goes through one such factor per join, and a sequence
// adds up hundreds of rows: the log takes `joins` of them back, from all but the largest term.
// Mean errors then lie within 2e-8 from 200 to 65536 columns (without: 5e-8 to 11e-8).
constexpr float kEx2Short = 5.0e-8f;
// Joins over 32 lanes and W warps: of the warps' sums one stays as it is.
constexpr float joins_of(int warps) { return 2.0f - 1.0f / (float)warps; }
// The log is that of the mantissa in fp32 (below 0.35 in magnitude, so good to 2^-25) and the
// exponent's in double: a thread does this once per row in front of a barrier, and the double
// log's chain of dependent steps took longer than a row of a few thousand columns.
ECO_DEV double token_logp(float raw_y, MaxSum a, double mul, float joins) {
  const int bits = __float_as_int(a.s) - 0x3f3504f3;  // mantissa in [sqrt 1/2, sqrt 2)
  const int e = bits >> 23;
  const float f = a.s > 0.0f && a.s < INFINITY ? __int_as_float((bits & 0x007fffff) + 0x3f3504f3) : a.s;
  const float small = logf(f) + kEx2Short * joins * (1.0f - __fdividef(1.0f, a.s));
  const double whole = a.s > 0.0f && a.s < INFINITY ? (double)e * 0.69314718055994530942 : 0.0;
  return ((double)raw_y - (double)a.m) * mul - (whole + (double)small);
}

// ------------------------------------------------ gradient from a coefficient per row
// A CTA writes one segment of one row (blockIdx.y: the segment), or one warp per short row.
template <typename T, int NT>
__global__ void __launch_bounds__(256)
    token_grad_kernel(const __grid_constant__ Rows R, const float2* __restrict__ stats,
                      const float* __restrict__ coef, const float* __restrict__ scale, float gain,
                      const __grid_constant__ Grad G, int64_t seg) {
  using GT = typename RowIo<T>::G;
  const float up = scale ? gain * *scale : gain;
  const int tid = threadIdx.x % NT;
  const int64_t v0 = (int64_t)blockIdx.y * seg;
  for (int64_t r = (int64_t)blockIdx.x * (blockDim.x / NT) + threadIdx.x / NT; r < R.rows;
       r += (int64_t)gridDim.x * (blockDim.x / NT)) {
    const T* x = static_cast<const T*>(R.x) + R.at(r, R.s0, R.s1);
    GT* g = static_cast<GT*>(G.g) + R.at(r, G.s0, G.s1);
    const float2 st = stats[r];
    const float k = st.y == 0.0f ? 0.0f : coef[r] * up;
    if (k == 0.0f)
      row_zero<T, NT>(x, g, R.cols, v0 + tid, v0 + seg);
    else
      row_grad<T, NT>(x, g, R.cols, Slope{st.x, R.c.hi, k * st.y, k, 0.0f}, R.tokens[r], v0 + tid, v0 + seg);
  }
}

// ------------------------------------------------ the policy loss
struct Policy {
  const float *old_logp, *adv, *ref;  // ref nullable
  float low, high, kl_coef;           // clip to [low, high]
  double denom;                       // > 0: given; else the count of rows that count, at least 1
};
struct Token {
  float loss, kl, coef;
  bool clipped;
};
// What a row's terms need besides its logits, loaded before they are needed.
struct Given {
  float old, adv, ref;
};
ECO_DEV Given given_of(const Policy& P, int64_t r) {
  return Given{P.old_logp[r], P.adv[r], P.ref ? P.ref[r] : 0.0f};
}
// free = -A r, held = -A clip(r); loss = max(free, held) + kl_coef kl; dloss/dlp.
ECO_DEV Token policy_token(const Policy& P, const Given& v, double lp) {
  const float A = v.adv;
  const float ratio = expf((float)(lp - (double)v.old));
  const float free = -A * ratio, held = -A * fminf(fmaxf(ratio, P.low), P.high);
  Token t;
  t.clipped = free < held;
  t.loss = t.clipped ? held : free;
  t.coef = t.clipped ? 0.0f : free;
  t.kl = 0.0f;
  if (P.ref) {
    const float d = (float)((double)v.ref - lp);
    const float e = expm1f(d);
    t.kl = e - d;
    t.loss += P.kl_coef * t.kl;
    t.coef -= P.kl_coef * e;
  }
  return t;
}

// How many rows count, at least 1, by the whole CTA.  Few rows: every CTA reads the masks
// itself (a few bytes per row from L2, against one launch more); many: from kCounts partial
// counts of a launch of its own.
constexpr int kCounts = 64;
constexpr int64_t kCountRows = 2048;  // more rows than this are counted beforehand

__global__ void __launch_bounds__(256) count_kernel(const __grid_constant__ Rows R, int* counts) {
  __shared__ int sh[8];
  int n = 0;
  for (int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x; r < R.rows; r += 256 * kCounts) n += R.counts(r);
  n = __reduce_add_sync(0xffffffffu, n);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = n;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 8; ++w) n += sh[w];
    counts[blockIdx.x] = n;
  }
}
ECO_DEV double policy_denom(const Rows& R, double given, const int* counts, int* sh) {
  if (given > 0.0) return given;
  int n = 0;
  if (counts) {
    for (int i = threadIdx.x; i < kCounts; i += blockDim.x) n += counts[i];
  } else {
    for (int64_t r = threadIdx.x; r < R.rows; r += blockDim.x) n += R.counts(r);
  }
  n = __reduce_add_sync(0xffffffffu, n);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = n;
  __syncthreads();
  int all = 0;
  for (int w = 0; w < (int)blockDim.x / 32; ++w) all += sh[w];
  __syncthreads();
  return all > 0 ? (double)all : 1.0;
}
// A coefficient over the denominator (its reciprocal, taken once), times the caller's factor.
ECO_DEV float over(float coef, double inv_denom, float gain) { return (float)((double)coef * inv_denom) * gain; }

struct Terms {  // per row: loss, kl, clipped
  float *loss, *kl, *clip;
};
ECO_DEV void put(const Terms& t, int64_t r, float loss, float kl, float clip) {
  t.loss[r] = loss;
  t.kl[r] = kl;
  t.clip[r] = clip;
}

// ------------------------------------------------ what a row leaves, and where rows lie
struct RowOut {  // what a row leaves besides its gradient; all nullable
  float* logp;
  double* lp64;
  float2* stats;
  float* coef0;
  Terms terms;
};
template <bool GRAD>
ECO_DEV void row_out(const RowOut& O, int64_t r, double lp, float2 st, const Token& t) {
  if (O.logp) O.logp[r] = (float)lp;
  if (O.lp64) O.lp64[r] = lp;
  if (O.stats) O.stats[r] = st;
  if (O.coef0) O.coef0[r] = 0.0f;
  if (GRAD) put(O.terms, r, t.loss, t.kl, t.clipped ? 1.0f : 0.0f);
}

// Offsets of every step-th row without a division per row.
struct Cursor {
  int r, i, n1, step, step_i;
  int64_t off, step_off, carry;
  ECO_DEV Cursor(const Rows& R, int first, int step_, int64_t s0, int64_t s1) {
    n1 = (int)R.n1;
    r = first;
    step = step_;
    const int o = n1 == (int)R.rows ? 0 : first / n1, so = n1 == (int)R.rows ? 0 : step / n1;
    i = first - o * n1;
    step_i = step - so * n1;
    off = o * s0 + i * s1;
    step_off = so * s0 + step_i * s1;
    carry = n1 == (int)R.rows ? 0 : s0 - n1 * s1;
  }
  ECO_DEV void next() {
    r += step;
    i += step_i;
    off += step_off;
    if (i >= n1) {
      i -= n1;
      off += carry;
    }
  }
};

// ------------------------------------------------ rows on NT threads
// Rows side by side in a CTA of 128 threads, or one row per CTA; as many CTAs per SM as registers
// allow, which is what hides a row's fixed work (the joins; one thread's logarithm and loss
// terms) and its loads' latency: nothing is copied ahead.  The gradient reads the row again, out
// of L1 or L2, where the rows in work (148 SMs x 1024 threads x 16 vectors: 39 MB) stay.
// Sixteen vectors per thread: with four or eight the fixed work is a larger share (bf16 65536 x
// 4096, us by 4 / 8 / 16: forward 131 / 109 / 92, policy loss 313 / 276 / 248; a ring of copies
// in shared memory, which leaves room for 16 warps only: 140 and 306).
constexpr int rows_beside(int nt) { return nt == 32 ? 4 : 1; }
constexpr int rows_ctas(int nt, bool grad) { return (grad ? 1024 : 1536) / (nt * rows_beside(nt)); }
template <typename T, int NT, bool GRAD>
__global__ void __launch_bounds__(NT * rows_beside(NT), rows_ctas(NT, GRAD))
    row_kernel(const __grid_constant__ Rows R, const __grid_constant__ Policy P, const int* counts, float gain,
               const __grid_constant__ RowOut O, const __grid_constant__ Grad G) {
  using GT = typename RowIo<T>::G;
  constexpr int E = RowIo<T>::E, W = NT / 32, BESIDE = rows_beside(NT);
  __shared__ MaxSum sh[W];
  __shared__ Slope row_sh[BESIDE];
  __shared__ int counts_sh[W * BESIDE];
  const int tid = threadIdx.x % NT, beside = threadIdx.x / NT, cols = (int)R.cols, rows = (int)R.rows;
  const double inv_denom = GRAD ? 1.0 / policy_denom(R, P.denom, counts, counts_sh) : 1.0;
  Cursor xc(R, (int)blockIdx.x * BESIDE + beside, (int)gridDim.x * BESIDE, R.s0, R.s1);
  Cursor gc(R, (int)blockIdx.x * BESIDE + beside, (int)gridDim.x * BESIDE, GRAD ? G.s0 : R.s0, GRAD ? G.s1 : R.s1);
  for (; xc.r < rows; xc.next(), gc.next()) {
    const T* x = static_cast<const T*>(R.x) + xc.off;
    const int y = R.counts(xc.r) ? (int)R.tokens[xc.r] : -1;
    const RowSplit sp = RowIo<T>::split(x, cols);
    const int vecs = (int)sp.vecs, edges = sp.head + sp.tail;
    const uint4* body = reinterpret_cast<const uint4*>(x + sp.head);
    float edge = -INFINITY, raw_y = 0.0f;
    Given v{0.0f, 0.0f, 0.0f};
    MaxSum a{-INFINITY, 0.0f};
    if (y >= 0) {
      if (tid < edges) edge = to_f32(x[sp.edge(tid, cols)]);
      if (tid == 0) {
        raw_y = to_f32(x[y]);
        if (GRAD) v = given_of(P, xc.r);
      }
      take_run<T, 4, false>(a, body + tid, NT, run_length<NT>(vecs, tid), R.c);
      if (tid < edges) {
        const float f[1] = {edge};
        take<1>(a, f, R.c);
      }
    }
    a = lanes_join<32>(a, R.c);
    if (W > 1) {
      if ((tid & 31) == 0) sh[tid >> 5] = a;
      __syncthreads();  // for rows that do not count too: the last row's slope has been read by all
      if (tid < 32) a = lanes_join<W>(sh[tid % W], R.c);
    }
    if (tid == 0) {
      double lp = 0.0;
      float inv = 0.0f, off = 0.0f, coef = 0.0f;
      Token t{0.0f, 0.0f, 0.0f, false};
      if (y >= 0) {
        lp = token_logp(raw_y, a, R.mul, joins_of(W));
        off = row_off(a.m);
        inv = 1.0f / a.s;
        if (GRAD) {
          t = policy_token(P, v, lp);
          coef = over(t.coef, inv_denom, gain);
        }
      }
      if (GRAD) row_sh[beside] = slope_of(off, R.c.hi, coef * inv, coef);
      row_out<GRAD>(O, xc.r, lp, make_float2(off, inv), t);
    }
    if (W > 1) __syncthreads(); else __syncwarp();  // row_sh; sh is free again
    if constexpr (GRAD) {
      const Slope c = row_sh[beside];
      GT* g = static_cast<GT*>(G.g) + gc.off;
      GT* gb = g + sp.head;
      const bool zero = y < 0 || c.coef == 0.0f;
      if (zero) {
        const float f[E] = {};
        for (int at = tid; at < vecs; at += NT) RowIo<T>::store(gb, at, f);
      } else {
        for (int at = tid; at < vecs; at += 4 * NT) {
          uint4 raw[4];
#pragma unroll
          for (int u = 0; u < 4; ++u)
            if (at + u * NT < vecs) raw[u] = __ldg(body + at + u * NT);
#pragma unroll
          for (int u = 0; u < 4; ++u)
            if (at + u * NT < vecs) store_slope<T, true>(gb, at + u * NT, raw[u], c);
        }
      }
      if (tid < edges) {
        const int j = (int)sp.edge(tid, cols);
        g[j] = from_f32<GT>(zero ? 0.0f : slope_at(edge, c, j == y));
      }
      const int yv = y - sp.head;  // the token's element, by the thread that has written its vector
      if (!zero && yv >= 0 && yv / E < vecs && yv / E % NT == tid) g[y] = from_f32<GT>(slope_at(to_f32(x[y]), c, true));
      if (W == 1) __syncwarp();  // row_sh is free again
    }
  }
}

// ------------------------------------------------ short rows
// The policy loss of rows that a warp holds in four vectors a lane: what counts is their fixed
// work, and here a warp has its next two rows on their way (cp.async by the lane that will use
// them, so no barrier belongs to the copies) while it does it (bf16 200000 x 1000: 322 us against
// 364 by the kernel above, int8 100000 x 1000: 192 against 208; of the bandwidth of a copy 0.38
// and 0.40).
//
// Vectors are counted from the 16-byte boundary at or before the row's start: the first and
// last may hold neighbours' elements, which are read (they share 16 bytes with the row) and
// left out.
constexpr int kPieces = 4;  // vectors per lane
constexpr int kRows = 3;    // rows in the ring

template <typename T>
__global__ void __launch_bounds__(32, 32)
    held_rows_kernel(const __grid_constant__ Rows R, const __grid_constant__ Policy P, const int* counts, float gain,
                     const __grid_constant__ RowOut O, const __grid_constant__ Grad G) {
  using GT = typename RowIo<T>::G;
  constexpr int E = RowIo<T>::E;
  __shared__ uint4 ring[kRows][kPieces][32];
  __shared__ Slope row_sh;
  __shared__ int counts_sh[1];
  const int lane = threadIdx.x, cols = (int)R.cols, rows = (int)R.rows, step = (int)gridDim.x;
  const double inv_denom = 1.0 / policy_denom(R, P.denom, counts, counts_sh);

  // A row on its way: its token (-1: it does not count) and the element its first vector
  // starts at (0 .. E - 1 before the row).
  struct Row {
    int y, skew;
  };
  Cursor xc(R, blockIdx.x, step, R.s0, R.s1);  // the next row to be issued
  // Its token and mask, loaded an iteration before they are looked at: no wait for them.
  int64_t token;
  bool kept;
  auto look = [&](int r) {
    token = -1;
    kept = false;
    if (r < rows) {
      token = R.tokens[r];
      kept = (!R.mask || R.mask[r]) && (!R.cu || (r >= R.cu[0] && r < R.cu[R.nseq]));
    }
  };
  auto issue = [&](int slot) {
    Row w{-1, 0};
    if (kept && token >= 0 && token < cols) {
      const T* x = static_cast<const T*>(R.x) + xc.off;
      w.y = (int)token;
      w.skew = (int)(reinterpret_cast<uintptr_t>(x) & 15) / (int)sizeof(T);
      const uint4* src = reinterpret_cast<const uint4*>(x - w.skew) + lane;
      const int left = (w.skew + cols + E - 1) / E - lane;  // vectors from mine on
      const uint32_t d = (uint32_t)__cvta_generic_to_shared(&ring[slot][0][lane]);
#pragma unroll
      for (int p = 0; p < kPieces; ++p)
        if (p * 32 < left)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d + p * 512), "l"(src + p * 32) : "memory");
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    xc.next();
    look(xc.r);
    return w;
  };
  // The row's vectors [first, whole) lie within it.  The elements before and behind them (fewer
  // than 2 E <= 32) go one to a lane, which loads them from the row itself: worked on in their
  // vectors, they would cost a lane E terms while the others wait.
  auto edge_index = [&](int skew) {
    const int end = skew + cols, head = skew > 0 ? min(E - skew, cols) : 0, tail = skew > 0 && end < E ? 0 : end % E;
    return lane < head ? lane : lane < head + tail ? cols - tail + lane - head : -1;
  };
  auto sum = [&](int slot, Row w, float edge) {
    MaxSum a{-INFINITY, 0.0f};
    if (w.y < 0) return a;
    const int first = w.skew > 0, end = w.skew + cols, whole = end / E - lane;
    const int pieces = (end / E + 31) / 32;
    auto group = [&](auto n) {  // a row of one or two pieces does not work on four
      constexpr int N = decltype(n)::value;
      uint4 raw[N];
      bool in[N];
#pragma unroll
      for (int p = 0; p < N; ++p) {
        in[p] = p * 32 < whole && p * 32 + lane >= first;
        raw[p] = ring[slot][p][lane];
      }
      take_vectors<T, false, N>(a, raw, in, R.c);
    };
    if (pieces == 1) group(std::integral_constant<int, 1>());
    else if (pieces == 2) group(std::integral_constant<int, 2>());
    else if (pieces > 2) group(std::integral_constant<int, 4>());
    if ((w.skew | cols % E) != 0) {
      const float f[1] = {edge};
      take<1>(a, f, R.c);
    }
    return a;
  };
  // What a row needs besides its vectors, loaded a row ahead.
  struct Beside {
    float raw_y, edge;
    Given v;
  };
  Cursor rc(R, blockIdx.x, step, R.s0, R.s1);
  auto beside = [&](Row w) {
    Beside b{0.0f, -INFINITY, Given{0.0f, 0.0f, 0.0f}};
    if (rc.r < rows && w.y >= 0) {
      const T* x = static_cast<const T*>(R.x) + rc.off;
      if (lane == 0) {
        b.raw_y = to_f32(x[w.y]);
        b.v = given_of(P, rc.r);
      }
      const int i = (w.skew | cols % E) != 0 ? edge_index(w.skew) : -1;
      if (i >= 0) b.edge = to_f32(x[i]);
    }
    rc.next();
    return b;
  };

  look(blockIdx.x);
  Cursor gc(R, blockIdx.x, step, G.s0, G.s1);  // the row in work
  Row w0 = issue(0), w1 = issue(1), w2 = issue(2);
  Beside b0 = beside(w0);
  for (int slot = 0; gc.r < rows; gc.next()) {
    const Beside b1 = beside(w1);
    asm volatile("cp.async.wait_group %0;" ::"n"(kRows - 1) : "memory");
    const MaxSum a = lanes_join<32>(sum(slot, w0, b0.edge), R.c);
    if (lane == 0) {
      double lp = 0.0;
      float inv = 0.0f, off = 0.0f, coef = 0.0f;
      Token t{0.0f, 0.0f, 0.0f, false};
      if (w0.y >= 0) {
        lp = token_logp(b0.raw_y, a, R.mul, joins_of(1));
        off = row_off(a.m);
        inv = 1.0f / a.s;
        t = policy_token(P, b0.v, lp);
        coef = over(t.coef, inv_denom, gain);
      }
      row_sh = slope_of(off, R.c.hi, coef * inv, coef);
      row_out<true>(O, gc.r, lp, make_float2(off, inv), t);
    }
    __syncwarp();
    const Slope c = row_sh;
    GT* g = static_cast<GT*>(G.g) + gc.off;
    // a row that does not count was not looked at: its gradient starts as its logits do
    const int skew = (int)((reinterpret_cast<uintptr_t>(g) / sizeof(GT)) & (E - 1));
    const bool zero = w0.y < 0 || c.coef == 0.0f;
    const int first = skew > 0, end = skew + cols, whole = end / E - lane;
    GT* gv = g - skew + lane * E;
    if (zero) {
      const float f[E] = {};
#pragma unroll
      for (int p = 0; p < kPieces; ++p)
        if (p * 32 < whole && p * 32 + lane >= first) RowIo<T>::store(gv, p * 32, f);
    } else {
#pragma unroll
      for (int p = 0; p < kPieces; ++p)
        if (p * 32 < whole && p * 32 + lane >= first) store_slope<T, true>(gv, p * 32, ring[slot][p][lane], c);
    }
    if ((skew | cols % E) != 0) {
      const int i = edge_index(skew);
      if (i >= 0) g[i] = from_f32<GT>(zero ? 0.0f : slope_at(b0.edge, c, i == w0.y));
    }
    const int yv = (w0.y + skew) / E;  // the token's element, by the lane that has written its vector
    if (!zero && yv >= first && yv < end / E && yv % 32 == lane) {
      const float xy = to_f32(reinterpret_cast<const T*>(&ring[slot][yv / 32][lane])[(w0.y + skew) % E]);
      g[w0.y] = from_f32<GT>(slope_at(xy, c, true));
    }
    __syncwarp();  // row_sh is free again
    w0 = w1, w1 = w2, w2 = issue(slot);
    b0 = b1;
    slot = slot == kRows - 1 ? 0 : slot + 1;
  }
}

// ------------------------------------------------ wide rows
// The whole policy loss.  The first kPlaces vectors per thread of a row stay in shared memory, the
// rest is read again for the gradient, from L2: the launch lets no more rows be in work than L2
// holds the rests of.  As soon as a place has been used for the last time, the next row's vector
// is copied there (cp.async by the thread that will use it), so memory is read while the end of a
// row is summed, joined and written.
// One read and one write of bf16 8192 x 131072: 815 us, 0.80 of the bandwidth of a copy (fp32 4096
// rows: 810, 0.81).  Reads are 9% above the logits' size (what L2 loses of the rests), the issue
// slots busy for 0.58 of the time; two CTAs per SM take turns at reading and writing.
constexpr int kPlaces = 12;
constexpr int kBatch = 4;  // vectors read again at a time

template <typename T, int NT>
__global__ void __launch_bounds__(NT, 1024 / NT)
    wide_rows_kernel(const __grid_constant__ Rows R, const __grid_constant__ Policy P, const int* counts, float gain,
                     const __grid_constant__ RowOut O, const __grid_constant__ Grad G) {
  using GT = typename RowIo<T>::G;
  using Io = RowIo<T>;
  constexpr int E = Io::E, W = NT / 32;
  extern __shared__ __align__(16) uint4 places[];  // [kPlaces][NT]
  __shared__ MaxSum sh[W];
  __shared__ Slope row_sh;
  __shared__ int counts_sh[W];
  const int tid = threadIdx.x, cols = (int)R.cols, rows = (int)R.rows, step = (int)gridDim.x;
  const double inv_denom = 1.0 / policy_denom(R, P.denom, counts, counts_sh);
  uint4* const mine = places + tid;
  const uint32_t mine_s = (uint32_t)__cvta_generic_to_shared(mine);
  Cursor xc(R, blockIdx.x, step, R.s0, R.s1);  // one row ahead of gc after the first fill
  Cursor gc(R, blockIdx.x, step, G.s0, G.s1);
  int64_t token = -1;
  bool kept = false;
  auto look = [&](int r) {  // loads only; looked at when the row's copies start
    token = -1;
    kept = false;
    if (r < rows) {
      token = R.tokens[r];
      kept = (!R.mask || R.mask[r]) && (!R.cu || (r >= R.cu[0] && r < R.cu[R.nseq]));
    }
  };
  struct Row {
    const T* x;
    int y, vecs, head;
  };
  auto next_row = [&]() {  // the row xc stands at
    Row w{static_cast<const T*>(R.x) + xc.off, -1, 0, 0};
    if (kept && token >= 0 && token < cols) {
      const RowSplit sp = Io::split(w.x, cols);
      w.y = (int)token;
      w.vecs = (int)sp.vecs;
      w.head = sp.head;
    }
    return w;
  };
  // These are read once: they leave L2 to the rests, of which a third was lost to them (fp32 4096
  // rows of 131072: 866 -> 804 us).
  uint64_t once;
  asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(once));
  auto copy = [&](const Row& w, int p) {
    if (p * NT + tid < w.vecs)
      asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(mine_s + p * NT * 16),
                   "l"(reinterpret_cast<const uint4*>(w.x + w.head) + p * NT + tid), "l"(once)
                   : "memory");
  };
  look(xc.r);
  Row w = next_row();
#pragma unroll
  for (int p = 0; p < kPlaces; ++p) copy(w, p);
  asm volatile("cp.async.commit_group;" ::: "memory");
  xc.next();
  look(xc.r);
  for (; gc.r < rows; gc.next()) {
    const int tail = cols - w.head - w.vecs * E, edges = w.y < 0 ? 0 : w.head + tail;
    const T* body = w.x + w.head;
    float raw_y = 0.0f, edge = 0.0f;
    Given v{0.0f, 0.0f, 0.0f};
    const int edge_at = tid < w.head ? tid : cols - tail + tid - w.head;
    if (w.y >= 0) {
      if (tid == 0) {
        raw_y = to_f32(w.x[w.y]);
        v = given_of(P, gc.r);
      }
      if (tid < edges) edge = to_f32(w.x[edge_at]);
    }
    const Row nw = next_row();
    MaxSum a{-INFINITY, 0.0f};
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    if (w.y >= 0) {
      const int run = run_length<NT>(w.vecs, tid), here = run < kPlaces ? run : kPlaces;
      take_run<T, kBatch, true>(a, mine, NT, here, R.c);
      take_run<T, kBatch, false>(a, reinterpret_cast<const uint4*>(body) + kPlaces * NT + tid, NT, run - kPlaces, R.c);
      if (tid < edges) {
        const float f[1] = {edge};
        take<1>(a, f, R.c);
      }
    }
    xc.next();
    look(xc.r);
    a = lanes_join<32>(a, R.c);
    if ((tid & 31) == 0) sh[tid >> 5] = a;
    __syncthreads();
    if (tid < 32) {
      a = lanes_join<W>(sh[tid % W], R.c);
      if (tid == 0) {
        double lp = 0.0;
        float inv = 0.0f, off = 0.0f, coef = 0.0f;
        Token t{0.0f, 0.0f, 0.0f, false};
        if (w.y >= 0) {
          lp = token_logp(raw_y, a, R.mul, joins_of(W));
          off = row_off(a.m);
          inv = 1.0f / a.s;
          t = policy_token(P, v, lp);
          coef = over(t.coef, inv_denom, gain);
        }
        row_sh = slope_of(off, R.c.hi, coef * inv, coef);
        row_out<true>(O, gc.r, lp, make_float2(off, inv), t);
      }
    }
    __syncthreads();  // row_sh, and sh is free again
    {
      const Slope c = row_sh;
      GT* g = static_cast<GT*>(G.g) + gc.off;
      const bool zero = w.y < 0 || c.coef == 0.0f;
      // a row that does not count was not split: its gradient starts as its logits do
      const RowSplit sp = Io::split(w.x, cols);
      GT* gb = g + sp.head;
      const int vecs = (int)sp.vecs;
      const int run = run_length<NT>(vecs, tid);
      GT* gp = gb + tid * E;
      if (zero) {
        const float f[E] = {};
        for (int p = 0; p < run; ++p, gp += NT * E) Io::store(gp, 0, f);
#pragma unroll
        for (int p = 0; p < kPlaces; ++p) copy(nw, p);
        asm volatile("cp.async.commit_group;" ::: "memory");
      } else {
#pragma unroll
        for (int p = 0; p < kPlaces; ++p) {
          if (p < run) store_slope<T, true>(gp, p * NT, mine[p * NT], c);
          copy(nw, p);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        const uint4* xp = reinterpret_cast<const uint4*>(body) + kPlaces * NT + tid;
        gp += kPlaces * NT * E;
        for (int left = run - kPlaces; left > 0; left -= kBatch, xp += kBatch * NT, gp += kBatch * NT * E) {
          uint4 raw[kBatch];
#pragma unroll
          for (int p = 0; p < kBatch; ++p)
            if (p < left) raw[p] = __ldcs(xp + p * NT);
#pragma unroll
          for (int p = 0; p < kBatch; ++p) {
            if (p < left) store_slope<T, true>(gp, p * NT, raw[p], c);
          }
        }
      }
      if (tid < sp.head + sp.tail) {
        const int j = (int)sp.edge(tid, cols);
        g[j] = from_f32<GT>(zero ? 0.0f : slope_at(edge, c, j == w.y));
      }
      const int yv = w.y - sp.head;  // the token's element, by the thread that has written its vector
      if (!zero && yv >= 0 && yv / E < vecs && yv / E % NT == tid)
        g[w.y] = from_f32<GT>(slope_at(to_f32(w.x[w.y]), c, true));
    }
    w = nw;
  }
}

// N sums over a CTA in a fixed order, to every thread; sh: 32 N doubles.  The warps' sums are
// joined by shuffles as well: one after the other they took longer than all the rest for few rows.
template <int N>
ECO_DEV void cta_sums(double (&v)[N], double* sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = (int)blockDim.x / 32;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  if (lane == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) sh[i * 32 + warp] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = lane < warps ? sh[i * 32 + lane] : 0.0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  __syncthreads();
}

// loss, kl and clip fraction from the rows' terms (one CTA, fixed order, sums in double).
__global__ void __launch_bounds__(1024) policy_finish_kernel(const __grid_constant__ Rows R, const Terms terms,
                                                              double denom, const int* counts, float* out) {
  __shared__ double sh[3 * 32];
  __shared__ int counts_sh[32];
  const double n = policy_denom(R, denom, counts, counts_sh);
  double v[3] = {};
  for (int64_t r = threadIdx.x; r < R.rows; r += blockDim.x) {
    v[0] += terms.loss[r];
    v[1] += terms.kl[r];
    v[2] += terms.clip[r];
  }
  cta_sums(v, sh);
  if (threadIdx.x < 3) out[threadIdx.x] = (float)((threadIdx.x == 0 ? v[0] : threadIdx.x == 1 ? v[1] : v[2]) / n);
}

// The policy loss from log-probabilities: terms and coefficients (one CTA).
__global__ void __launch_bounds__(1024) policy_tokens_kernel(const __grid_constant__ Rows R,
                                                              const __grid_constant__ Policy P, const double* lp64,
                                                              float* coef, float* out) {
  __shared__ double sh[3 * 32];
  __shared__ int counts_sh[32];
  const double n = policy_denom(R, P.denom, nullptr, counts_sh), inv = 1.0 / n;
  double v[3] = {};
  for (int64_t r = threadIdx.x; r < R.rows; r += blockDim.x) {
    float k = 0.0f;
    if (R.counts(r)) {
      const Token t = policy_token(P, given_of(P, r), lp64[r]);
      v[0] += t.loss;
      v[1] += t.kl;
      v[2] += t.clipped ? 1.0 : 0.0;
      k = over(t.coef, inv, 1.0f);
    }
    coef[r] = k;
  }
  cta_sums(v, sh);
  if (threadIdx.x < 3) out[threadIdx.x] = (float)((threadIdx.x == 0 ? v[0] : threadIdx.x == 1 ? v[1] : v[2]) / n);
}

// ------------------------------------------------ the preference loss
struct Pairs {
  const float* ref;
  int64_t seq_len;  // rows per sequence when cu is null
  int64_t pairs;
  double beta, smooth, denom;
  int kind;
  bool average;
};

// One CTA per pair: both sequences' sums of lp - ref in double, the pair's loss and slope,
// the coefficients of its rows.
__global__ void __launch_bounds__(256) pair_kernel(const __grid_constant__ Rows R, const __grid_constant__ Pairs P,
                                                    const double* lp64, float* coef, float* log_ratio, float* margin,
                                                    double* pair_loss) {
  __shared__ double sh[4 * 32];
  const int64_t p = blockIdx.x;
  int64_t lo[2], hi[2];
  double ratio[2], per[2], v[4] = {};  // sums and numbers of rows
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const int64_t q = p + s * P.pairs;
    int64_t b = R.cu ? (int64_t)R.cu[q] : q * P.seq_len, e = R.cu ? (int64_t)R.cu[q + 1] : (q + 1) * P.seq_len;
    b = b < 0 ? 0 : (b > R.rows ? R.rows : b);
    e = e < b ? b : (e > R.rows ? R.rows : e);
    for (int64_t r = b + threadIdx.x; r < e; r += blockDim.x)
      if (R.counts(r)) {
        v[s] += lp64[r] - (double)P.ref[r];
        v[2 + s] += 1.0;
      }
    lo[s] = b;
    hi[s] = e;
  }
  cta_sums(v, sh);
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    per[s] = P.average && v[2 + s] > 0.0 ? 1.0 / v[2 + s] : 1.0;
    ratio[s] = v[s] * per[s];
  }
  const double delta = ratio[0] - ratio[1], h = P.beta * delta;
  double loss, slope;  // slope: d loss / d delta
  if (P.kind == ECO_PREFERENCE_SIGMOID) {
    const double far = log1p(exp(-fabs(h)));  // softplus(-|h|)
    loss = (1.0 - P.smooth) * (far + fmax(-h, 0.0)) + P.smooth * (far + fmax(h, 0.0));
    slope = P.beta * (1.0 / (1.0 + exp(-h)) - (1.0 - P.smooth));
  } else if (P.kind == ECO_PREFERENCE_HINGE) {
    loss = fmax(1.0 - h, 0.0);
    slope = h < 1.0 ? -P.beta : (h >= 1.0 ? 0.0 : h);
  } else {
    const double off = delta - 0.5 / P.beta;
    loss = off * off;
    slope = 2.0 * off;
  }
  if (threadIdx.x == 0) {
    log_ratio[p] = (float)ratio[0];
    log_ratio[p + P.pairs] = (float)ratio[1];
    margin[p] = (float)h;
    pair_loss[p] = loss;
  }
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const float k = (float)((s ? -slope : slope) * per[s] / P.denom);
    for (int64_t r = lo[s] + threadIdx.x; r < hi[s]; r += blockDim.x)
      if (R.counts(r)) coef[r] = k;
  }
}

__global__ void __launch_bounds__(256) pair_finish_kernel(const double* pair_loss, int64_t pairs, double denom,
                                                           float* out) {
  __shared__ double sh[32];
  double a[1] = {};
  for (int64_t p = threadIdx.x; p < pairs; p += blockDim.x) a[0] += pair_loss[p];
  cta_sums(a, sh);
  if (threadIdx.x == 0) out[0] = (float)(a[0] / denom);
}

// ------------------------------------------------ host side
Rows rows_of(const eco_logits_t& L, const int64_t* tokens, const uint8_t* mask, const int32_t* cu, int64_t nseq) {
  Rows R;
  R.x = L.x;
  R.rows = L.n0 * L.n1;
  R.n1 = L.n0 == 1 ? R.rows : L.n1;
  R.s0 = L.s0;
  R.s1 = L.s1;
  R.cols = L.cols;
  R.mul = L.mul;
  const double c = L.mul * 1.4426950408889634;
  R.c.hi = std::nextafter((float)c, 0.0f);  // below c: the rest is positive, and -inf times it is -inf
  if ((double)R.c.hi >= c) R.c.hi = std::nextafter(R.c.hi, 0.0f);
  R.c.lo = (float)(c - (double)R.c.hi);
  R.tokens = tokens;
  R.mask = mask;
  R.cu = cu;
  R.nseq = (int)nseq;
  return R;
}

// Threads of a kernel of one CTA over n rows.
unsigned one_cta(int64_t n) { return (unsigned)std::min<int64_t>(1024, (n + 31) / 32 * 32); }

int esize(int type) { return type == ECO_F32 ? 4 : type == ECO_I8 ? 1 : 2; }

int check_logits(const eco_logits_t* L, const int64_t* tokens, const char* who) {
  ECO_REQUIRE(L && L->n0 >= 0 && L->n1 >= 0 && L->cols > 0, ECO_ERR_ARG, "%s: bad shape", who);
  ECO_REQUIRE(L->type >= ECO_F32 && L->type <= ECO_I8, ECO_ERR_ARG, "%s: unknown logits type %d", who, L->type);
  ECO_REQUIRE(L->n0 == 0 || L->n1 == 0 || (L->x && tokens), ECO_ERR_ARG, "%s: null logits or tokens", who);
  ECO_REQUIRE(L->mul >= 1e-30 && L->mul <= 1e30, ECO_ERR_ARG, "%s: the logits' factor must lie in [1e-30, 1e30]", who);
  ECO_REQUIRE(L->s0 >= 0 && L->s1 >= 0, ECO_ERR_ARG, "%s: negative strides", who);
  ECO_REQUIRE(reinterpret_cast<uintptr_t>(L->x) % (uintptr_t)esize(L->type) == 0, ECO_ERR_MISALIGNED,
              "%s: logits are not aligned to their type", who);
  // 2^30, so that a row's number and a step of the grid more stay below 2^31
  ECO_REQUIRE(L->n1 == 0 || L->n0 <= ((int64_t)1 << 30) / L->n1, ECO_ERR_ARG, "%s: more than 2^30 rows", who);
  ECO_REQUIRE(L->cols <= (int64_t)1 << 28, ECO_ERR_ARG, "%s: more than 2^28 columns", who);
  return ECO_OK;
}

// A 16-byte vector of logits and the vector of as many gradient elements hold the same
// elements: every gradient row starts as many elements behind such a boundary as its logits row.
int check_grad(const eco_logits_t& L, const eco_grad_t* G, const char* who) {
  ECO_REQUIRE(G && G->g && G->s0 >= 0 && G->s1 >= 0 && (L.n1 <= 1 || G->s1 >= L.cols) &&
                  (L.n0 <= 1 || G->s0 >= L.cols),
              ECO_ERR_ARG, "%s: bad gradient layout", who);
  const int64_t es = esize(L.type), ges = es == 1 ? 4 : es, per = 16 / es;
  const int64_t xb = (int64_t) reinterpret_cast<uintptr_t>(L.x), gb = (int64_t) reinterpret_cast<uintptr_t>(G->g);
  ECO_REQUIRE(gb % ges == 0 && (gb / ges - xb / es) % per == 0 && (L.n0 <= 1 || (G->s0 - L.s0) % per == 0) &&
                  (L.n1 <= 1 || (G->s1 - L.s1) % per == 0),
              ECO_ERR_MISALIGNED, "%s: gradient rows must start like the logits rows, modulo %d elements", who,
              (int)per);
  return ECO_OK;
}

template <typename F>
int by_type(int type, F f) {
  switch (type) {
    case ECO_F32: return f((float*)nullptr);
    case ECO_BF16: return f((__nv_bfloat16*)nullptr);
    case ECO_F16: return f((__half*)nullptr);
    default: return f((int8_t*)nullptr);
  }
}

// Vectors of a row, at whatever alignment it starts.
template <typename T>
int64_t row_vecs(const Rows& R) {
  constexpr int64_t E = RowIo<T>::E;
  const bool on_16 = eco_aligned16(R.x) && (R.rows == R.n1 || R.s0 % E == 0) && (R.n1 <= 1 || R.s1 % E == 0);
  return (R.cols + (on_16 ? 0 : E - 1) + E - 1) / E;
}

// walk: resident CTAs that walk down the rows; else one CTA after the other.
template <typename T, int NT, bool GRAD>
void launch_row(bool walk, const Rows& R, const Policy& P, const int* counts, float gain, const RowOut& O,
                const Grad& G, cudaStream_t s) {
  const int64_t most = walk ? (int64_t)eco_num_sms() * rows_ctas(NT, GRAD) : 1 << 20;
  const int64_t grid = std::min<int64_t>((R.rows + rows_beside(NT) - 1) / rows_beside(NT), most);
  row_kernel<T, NT, GRAD><<<(unsigned)grid, NT * rows_beside(NT), 0, s>>>(R, P, counts, gain, O, G);
}
// Threads of a row by its vectors: one per sixteen of them (eight of int8 where a gradient of
// four times their size is written: 32768 x 8192 254 us against 288), one per four where the rows
// would otherwise leave most of the SMs' threads without work (bf16 1 to 148 rows of 8192: 2.6 to
// 2.9 us against 3.6 to 3.9; 1500 rows: 7.7 against 7.2).
template <typename T, bool GRAD>
void by_rows(int64_t vecs, const Rows& R, const Policy& P, const int* counts, float gain, const RowOut& O,
             const Grad& G, cudaStream_t s) {
  int64_t per = GRAD && sizeof(T) == 1 ? 8 : 16;
  if (R.rows * (vecs / per) < (int64_t)eco_num_sms() * 512) per = 4;
  // The gradient needs the number of rows that count.  Where every CTA counts them itself, few CTAs
  // walk; where that is done, they walk if a row is soon over (fp32 131072 x 1024: 241 us against
  // 261; bf16 32768 x 8192: 237 against 228, the next row's loads then start earlier).
  const bool walk = GRAD && (vecs <= 256 || !(counts || P.denom > 0.0));
  if (vecs <= 32 * per) launch_row<T, 32, GRAD>(walk, R, P, counts, gain, O, G, s);
  else if (vecs <= 64 * per) launch_row<T, 64, GRAD>(walk, R, P, counts, gain, O, G, s);
  else if (vecs <= 128 * per) launch_row<T, 128, GRAD>(walk, R, P, counts, gain, O, G, s);
  else if (vecs <= 256 * per) launch_row<T, 256, GRAD>(walk, R, P, counts, gain, O, G, s);
  else launch_row<T, 512, GRAD>(walk, R, P, counts, gain, O, G, s);
}

template <typename T, int NT>
bool launch_wide(const Rows& R, const Policy& P, const int* counts, float gain, const RowOut& O, const Grad& G,
                 cudaStream_t s) {
  const auto kernel = wide_rows_kernel<T, NT>;
  constexpr int smem = kPlaces * NT * 16;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return false;
  const int64_t grid = std::min<int64_t>(R.rows, (int64_t)eco_num_sms() * (1024 / NT));
  kernel<<<(unsigned)grid, NT, smem, s>>>(R, P, counts, gain, O, G);
  return true;
}
// Wider rows than this (in vectors) go to the kernel that keeps their first part on the chip: bf16
// 8192 x 32768, 4096 vectors, 247 us by either; 8192 x 131072 818 us against 960.
constexpr int64_t kRowVecs = 4096;
// Whether what the rows in work leave to L2 fits there: half of its 126 MB, since either die
// keeps its own copy of what its SMs read.
bool rests_fit(int64_t vecs, int threads) {
  const int64_t rest = std::max<int64_t>(0, vecs - (int64_t)kPlaces * threads) * 16;
  return rest * eco_num_sms() * (1024 / threads) <= (int64_t)56 << 20;
}

template <typename T>
void launch_grad(const Rows& R, const float2* stats, const float* coef, const float* scale, float gain,
                 const Grad& G, cudaStream_t s) {
  const int64_t vecs = R.cols / RowIo<T>::E + 1;
  // A warp per row of up to 512 vectors (bf16 65536 x 4096: 171 us, 0.96 of the bandwidth of a
  // copy; a CTA of 256 threads per row, two vectors each: 213), 128 where there are few rows.
  if (vecs <= (R.rows >= 8 * (int64_t)eco_num_sms() ? 513 : 129)) {
    const int64_t grid = std::min<int64_t>((R.rows + 7) / 8, 1 << 20);
    token_grad_kernel<T, 32><<<(unsigned)grid, 256, 0, s>>>(R, stats, coef, scale, gain, G, INT64_MAX / 2);
  } else {
    // segments of 2048 vectors (32 KB of logits), eight loads of each thread
    const int64_t seg = 2048;
    const dim3 grid((unsigned)std::min<int64_t>(R.rows, 1 << 20), (unsigned)((vecs + seg - 1) / seg));
    token_grad_kernel<T, 256><<<grid, 256, 0, s>>>(R, stats, coef, scale, gain, G, seg);
  }
}

}  // namespace

extern "C" int eco_token_logp(const eco_logits_t* logits, const int64_t* tokens, const uint8_t* mask,
                              const int32_t* cu_seqlens, int64_t num_seqs, float* logp, double* logp64,
                              float* row_stats, float* coef_zero, eco_stream_t stream) {
  if (int rc = check_logits(logits, tokens, "eco_token_logp")) return rc;
  ECO_REQUIRE(!cu_seqlens || num_seqs > 0, ECO_ERR_ARG, "eco_token_logp: no sequences");
  const Rows R = rows_of(*logits, tokens, mask, cu_seqlens, num_seqs);
  if (R.rows == 0) return ECO_OK;
  ECO_REQUIRE(logp || logp64, ECO_ERR_ARG, "eco_token_logp: no output");
  float2* st = reinterpret_cast<float2*>(row_stats);
  by_type(logits->type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    const RowOut O{logp, logp64, st, coef_zero, Terms{}};
    by_rows<T, false>(row_vecs<T>(R), R, Policy{}, nullptr, 0.0f, O, Grad{}, eco_stream(stream));
    return 0;
  });
  return eco_launch_check("eco_token_logp");
}

extern "C" int eco_token_grad(const eco_logits_t* logits, const int64_t* tokens, const float* row_stats,
                              const float* coef, const float* scale, double gain, const eco_grad_t* grad,
                              eco_stream_t stream) {
  if (int rc = check_logits(logits, tokens, "eco_token_grad")) return rc;
  const Rows R = rows_of(*logits, tokens, nullptr, nullptr, 0);
  if (R.rows == 0) return ECO_OK;
  ECO_REQUIRE(row_stats && coef, ECO_ERR_ARG, "eco_token_grad: null row statistics or coefficients");
  if (int rc = check_grad(*logits, grad, "eco_token_grad")) return rc;
  const Grad G{grad->g, grad->s0, grad->s1};
  by_type(logits->type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    launch_grad<T>(R, reinterpret_cast<const float2*>(row_stats), coef, scale, (float)gain, G, eco_stream(stream));
    return 0;
  });
  return eco_launch_check("eco_token_grad");
}

static int policy_of(Policy& P, const float* old_logp, const float* adv, const float* ref, double low, double high,
                     double kl_coef, double denom, const char* who) {
  ECO_REQUIRE(old_logp && adv, ECO_ERR_ARG, "%s: null old log-probabilities or advantages", who);
  ECO_REQUIRE(low >= 0.0 && high >= low && std::isfinite(kl_coef) && !std::isnan(denom), ECO_ERR_ARG,
              "%s: bad clip range or coefficients", who);
  P = Policy{old_logp, adv, ref, (float)low, (float)high, (float)kl_coef, denom};
  return ECO_OK;
}

extern "C" int eco_policy_grad(const eco_logits_t* logits, const int64_t* tokens, const uint8_t* mask,
                               const float* old_logp, const float* adv, const float* ref_logp, double low,
                               double high, double kl_coef, double denom, double gain, float* logp, float* terms,
                               float* out, const eco_grad_t* grad, eco_stream_t stream) {
  if (int rc = check_logits(logits, tokens, "eco_policy_grad")) return rc;
  ECO_REQUIRE(out, ECO_ERR_ARG, "eco_policy_grad: null output");
  const Rows R = rows_of(*logits, tokens, mask, nullptr, 0);
  cudaStream_t s = eco_stream(stream);
  if (R.rows == 0) {
    if (cudaMemsetAsync(out, 0, 3 * sizeof(float), s) != cudaSuccess) return eco_launch_check("eco_policy_grad");
    return ECO_OK;
  }
  Policy P;
  if (int rc = policy_of(P, old_logp, adv, ref_logp, low, high, kl_coef, denom, "eco_policy_grad")) return rc;
  ECO_REQUIRE(logp && terms, ECO_ERR_ARG, "eco_policy_grad: null output");
  if (int rc = check_grad(*logits, grad, "eco_policy_grad")) return rc;
  const Grad G{grad->g, grad->s0, grad->s1};
  const Terms t{terms, terms + R.rows, terms + 2 * R.rows};
  int* counts = nullptr;
  if (!(denom > 0.0) && R.rows > kCountRows) {
    counts = reinterpret_cast<int*>(terms + 3 * R.rows);
    count_kernel<<<kCounts, 256, 0, s>>>(R, counts);
  }
  bool ok = true;
  by_type(logits->type, [&](auto* p) {
    using T = std::remove_pointer_t<decltype(p)>;
    const int64_t vecs = row_vecs<T>(R);
    const RowOut O{logp, nullptr, nullptr, nullptr, t};
    if (vecs <= 32 * kPieces)
      held_rows_kernel<T><<<(unsigned)std::min<int64_t>(R.rows, (int64_t)eco_num_sms() * 32), 32, 0, s>>>(
          R, P, counts, (float)gain, O, G);
    else if (vecs <= kRowVecs)
      by_rows<T, true>(vecs, R, P, counts, (float)gain, O, G, s);
    else
      ok = rests_fit(vecs, 512) ? launch_wide<T, 512>(R, P, counts, (float)gain, O, G, s)
                                : launch_wide<T, 1024>(R, P, counts, (float)gain, O, G, s);
    return 0;
  });
  if (!ok) return eco_fail(ECO_ERR_LAUNCH, "eco_policy_grad: %s", cudaGetErrorString(cudaGetLastError()));
  policy_finish_kernel<<<1, one_cta(R.rows), 0, s>>>(R, t, denom, counts, out);
  return eco_launch_check("eco_policy_grad");
}

extern "C" int eco_policy_forward(const eco_logits_t* logits, const int64_t* tokens, const uint8_t* mask,
                                  const float* old_logp, const float* adv, const float* ref_logp, double low,
                                  double high, double kl_coef, double denom, float* logp, double* logp64,
                                  float* row_stats, float* coef, float* out, eco_stream_t stream) {
  if (int rc = check_logits(logits, tokens, "eco_policy_forward")) return rc;
  ECO_REQUIRE(out, ECO_ERR_ARG, "eco_policy_forward: null output");
  const Rows R = rows_of(*logits, tokens, mask, nullptr, 0);
  cudaStream_t s = eco_stream(stream);
  if (R.rows == 0) {
    if (cudaMemsetAsync(out, 0, 3 * sizeof(float), s) != cudaSuccess) return eco_launch_check("eco_policy_forward");
    return ECO_OK;
  }
  Policy P;
  if (int rc = policy_of(P, old_logp, adv, ref_logp, low, high, kl_coef, denom, "eco_policy_forward")) return rc;
  ECO_REQUIRE(logp64 && row_stats && coef, ECO_ERR_ARG, "eco_policy_forward: null output");
  if (int rc = eco_token_logp(logits, tokens, mask, nullptr, 0, logp, logp64, row_stats, nullptr, stream)) return rc;
  policy_tokens_kernel<<<1, one_cta(R.rows), 0, s>>>(R, P, logp64, coef, out);
  return eco_launch_check("eco_policy_forward");
}

extern "C" int eco_preference(const eco_logits_t* logits, const int64_t* tokens, const uint8_t* mask,
                              const float* ref_logp, const int32_t* cu_seqlens, int64_t seq_len, int64_t pairs,
                              int kind, double beta, double label_smoothing, int average, double denom, double gain,
                              double* wide, float* row_stats, float* coef, float* log_ratio, float* margin,
                              float* loss, const eco_grad_t* grad, eco_stream_t stream) {
  if (int rc = check_logits(logits, tokens, "eco_preference")) return rc;
  const Rows R = rows_of(*logits, tokens, mask, cu_seqlens, 2 * pairs);
  ECO_REQUIRE(pairs > 0 && pairs < (1 << 30) && seq_len >= 0 && wide && log_ratio && margin && loss &&
                  (R.rows == 0 || (ref_logp && row_stats && coef)),
              ECO_ERR_ARG, "eco_preference: bad arguments");
  ECO_REQUIRE(cu_seqlens || R.rows / 2 / pairs >= seq_len, ECO_ERR_ARG, "eco_preference: more sequences than rows");
  ECO_REQUIRE(kind >= ECO_PREFERENCE_SIGMOID && kind <= ECO_PREFERENCE_IPO, ECO_ERR_ARG,
              "eco_preference: unknown kind %d", kind);
  ECO_REQUIRE(std::isfinite(beta) && beta > 0.0 && label_smoothing >= 0.0 && label_smoothing <= 1.0 && denom > 0.0,
              ECO_ERR_ARG, "eco_preference: bad beta, smoothing or denominator");
  if (grad && R.rows > 0)
    if (int rc = check_grad(*logits, grad, "eco_preference")) return rc;
  const Pairs P{ref_logp, seq_len, pairs, beta, label_smoothing, denom, kind, average != 0};
  cudaStream_t s = eco_stream(stream);
  if (R.rows > 0)
    if (int rc = eco_token_logp(logits, tokens, mask, cu_seqlens, 2 * pairs, nullptr, wide, row_stats, coef, stream))
      return rc;
  pair_kernel<<<(unsigned)pairs, 256, 0, s>>>(R, P, wide, coef, log_ratio, margin, wide + R.rows);
  pair_finish_kernel<<<1, std::min(256u, one_cta(pairs)), 0, s>>>(wide + R.rows, pairs, denom, loss);
  if (int rc = eco_launch_check("eco_preference")) return rc;
  return grad ? eco_token_grad(logits, tokens, row_stats, coef, nullptr, gain, grad, stream) : ECO_OK;
}
