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
// Sums are fp32 per thread over its share of the row and joined in a fixed order; the log
// of the sum and the token's term are taken in double, once per row, because
// exp(ref - lp) - (ref - lp) - 1 loses what fp32 loses twice over.
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

// What is subtracted before the exponential: m, and 0 for -inf alone (whose terms are then 0).
// x - m comes first and is multiplied after: a row masked to its type's lowest value would
// leave the fp32 range as x * c, and as x - m is 0 or -inf.
ECO_DEV float row_off(float m) { return m == -INFINITY ? 0.0f : m; }
ECO_DEV float term(float x, float off, float c) { return ex2((x - off) * c); }

struct MaxSum {
  float m, s;
};
ECO_DEV MaxSum join(MaxSum a, MaxSum b, float c) {
  const float m = fmaxf(a.m, b.m);
  const float off = row_off(m);
  return MaxSum{m, a.s * term(a.m, off, c) + b.s * term(b.m, off, c)};
}

template <int E>
ECO_DEV void take(MaxSum& a, const float (&x)[E], float c) {
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

// Joined over the NT threads of a row; every thread gets the same bits.
template <int NT>
ECO_DEV MaxSum row_join(MaxSum a, float c, MaxSum* sh) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    MaxSum b;
    b.m = __shfl_xor_sync(0xffffffffu, a.m, o);
    b.s = __shfl_xor_sync(0xffffffffu, a.s, o);
    a = (threadIdx.x & o) ? join(b, a, c) : join(a, b, c);
  }
  if (NT > 32) {
    constexpr int W = NT / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) sh[warp] = a;
    __syncthreads();
    a = sh[lane % W];
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) {
      MaxSum b;
      b.m = __shfl_xor_sync(0xffffffffu, a.m, o);
      b.s = __shfl_xor_sync(0xffffffffu, a.s, o);
      a = (lane & o) ? join(b, a, c) : join(a, b, c);
    }
  }
  return a;
}

template <typename T, int NT>
ECO_DEV MaxSum row_stats(const T* x, int64_t cols, float c, int tid, MaxSum* sh) {
  constexpr int E = RowIo<T>::E;
  const RowSplit sp = RowIo<T>::split(x, cols);
  MaxSum a{-INFINITY, 0.0f};
  const T* body = x + sp.head;
  int64_t v = tid;
  for (; v + 3 * NT < sp.vecs; v += 4 * NT) {
    typename RowIo<T>::Raw r[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) r[u] = RowIo<T>::load(body, v + u * NT);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      float f[E];
      RowIo<T>::unpack(r[u], f);
      take<E>(a, f, c);
    }
  }
  for (; v < sp.vecs; v += NT) {
    float f[E];
    RowIo<T>::unpack(RowIo<T>::load(body, v), f);
    take<E>(a, f, c);
  }
  if (tid < sp.head + sp.tail) {
    const float f[1] = {to_f32(x[sp.edge(tid, cols)])};
    take<1>(a, f, c);
  }
  return row_join<NT>(a, c, sh);
}

// g_j = -k 2^((x_j - off) c) (+ coef at y)
template <typename T, int NT>
ECO_DEV void row_grad(const T* x, typename RowIo<T>::G* g, int64_t cols, float c, float off, float k, float coef,
                      int64_t y, int64_t tid, int64_t v_end) {
  constexpr int E = RowIo<T>::E;
  const RowSplit sp = RowIo<T>::split(x, cols);
  const T* body = x + sp.head;
  typename RowIo<T>::G* gb = g + sp.head;
  const int64_t yb = y - sp.head;
  const int64_t vend = v_end < sp.vecs ? v_end : sp.vecs;
  for (int64_t v0 = tid; v0 < vend; v0 += 4 * NT) {
    typename RowIo<T>::Raw r[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (v0 + u * NT < vend) r[u] = RowIo<T>::load_last(body, v0 + u * NT);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t v = v0 + u * NT;
      if (v >= vend) break;
      float f[E];
      RowIo<T>::unpack(r[u], f);
#pragma unroll
      for (int i = 0; i < E; ++i) f[i] = -k * term(f[i], off, c);
      const int64_t d = yb - v * E;
      if (d >= 0 && d < E) {
#pragma unroll
        for (int i = 0; i < E; ++i)
          if (d == i) f[i] += coef;
      }
      RowIo<T>::store(gb, v, f);
    }
  }
  if (tid < sp.head + sp.tail) {  // the threads of the row's first segment
    const int64_t j = sp.edge((int)tid, cols);
    const float f = -k * term(to_f32(x[j]), off, c) + (j == y ? coef : 0.0f);
    g[j] = from_f32<typename RowIo<T>::G>(f);
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
  float c;  // mul * log2 e
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

// The row's term in double: (raw_y - m) mul - log s.
ECO_DEV double token_logp(float raw_y, MaxSum a, double mul) {
  return ((double)raw_y - (double)a.m) * mul - log((double)a.s);
}

// ------------------------------------------------ forward: lp and what the gradient needs
// One warp per row for short rows, one CTA per row for long ones.
template <typename T, int NT>
__global__ void __launch_bounds__(NT < 256 ? 256 : NT)
    token_logp_kernel(const __grid_constant__ Rows R, float* logp, double* lp64, float2* stats, float* coef0) {
  __shared__ MaxSum sh[NT > 32 ? NT / 32 : 1];
  const int tid = threadIdx.x % NT;
  for (int64_t r = (int64_t)blockIdx.x * (blockDim.x / NT) + threadIdx.x / NT; r < R.rows;
       r += (int64_t)gridDim.x * (blockDim.x / NT)) {
    const bool counts = R.counts(r);
    double lp = 0.0;
    float2 st = make_float2(0.0f, 0.0f);
    if (counts) {
      const T* x = static_cast<const T*>(R.x) + R.at(r, R.s0, R.s1);
      const float raw_y = tid == 0 ? to_f32(x[R.tokens[r]]) : 0.0f;
      const MaxSum a = row_stats<T, NT>(x, R.cols, R.c, tid, sh);
      if (tid == 0) {
        lp = token_logp(raw_y, a, R.mul);
        st = make_float2(row_off(a.m), 1.0f / a.s);
      }
      if (NT > 32) __syncthreads();  // sh is free again
    }
    if (tid == 0) {
      if (logp) logp[r] = (float)lp;
      if (lp64) lp64[r] = lp;
      if (stats) stats[r] = st;
      if (coef0) coef0[r] = 0.0f;
    }
  }
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
      row_grad<T, NT>(x, g, R.cols, R.c, st.x, k * st.y, k, R.tokens[r], v0 + tid, v0 + seg);
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
// free = -A r, held = -A clip(r); loss = max(free, held) + kl_coef kl; dloss/dlp.
ECO_DEV Token policy_token(const Policy& P, int64_t r, double lp) {
  const float A = P.adv[r];
  const float ratio = expf((float)(lp - (double)P.old_logp[r]));
  const float free = -A * ratio, held = -A * fminf(fmaxf(ratio, P.low), P.high);
  Token t;
  t.clipped = free < held;
  t.loss = t.clipped ? held : free;
  t.coef = t.clipped ? 0.0f : free;
  t.kl = 0.0f;
  if (P.ref) {
    const float d = (float)((double)P.ref[r] - lp);
    const float e = expm1f(d);
    t.kl = e - d;
    t.loss += P.kl_coef * t.kl;
    t.coef -= P.kl_coef * e;
  }
  return t;
}

// How many rows count, at least 1, by the whole CTA (every CTA reads the masks itself: a few
// bytes per row from L2, against one launch more).
ECO_DEV double policy_denom(const Rows& R, double given, int* sh) {
  if (given > 0.0) return given;
  int n = 0;
  for (int64_t r = threadIdx.x; r < R.rows; r += blockDim.x) n += R.counts(r);
  n = __reduce_add_sync(0xffffffffu, n);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = n;
  __syncthreads();
  int all = 0;
  for (int w = 0; w < (int)blockDim.x / 32; ++w) all += sh[w];
  __syncthreads();
  return all > 0 ? (double)all : 1.0;
}

struct Terms {  // per row: loss, kl, clipped
  float *loss, *kl, *clip;
};
ECO_DEV void put(const Terms& t, int64_t r, float loss, float kl, float clip) {
  t.loss[r] = loss;
  t.kl[r] = kl;
  t.clip[r] = clip;
}

// The whole policy loss of a row: statistics, coefficient, gradient.  The second pass finds
// the row in L2 (148 SMs x rows in flight of up to 512 KB against 126 MB).
template <typename T, int NT>
__global__ void __launch_bounds__(NT < 256 ? 256 : NT)
    policy_row_kernel(const __grid_constant__ Rows R, const __grid_constant__ Policy P, float gain, float* logp,
                      const __grid_constant__ Terms terms, const __grid_constant__ Grad G) {
  using GT = typename RowIo<T>::G;
  __shared__ MaxSum sh[NT > 32 ? NT / 32 : 1];
  __shared__ int counts_sh[32];
  __shared__ float coef_sh;
  const double denom = policy_denom(R, P.denom, counts_sh);
  const int tid = threadIdx.x % NT;
  for (int64_t r = (int64_t)blockIdx.x * (blockDim.x / NT) + threadIdx.x / NT; r < R.rows;
       r += (int64_t)gridDim.x * (blockDim.x / NT)) {
    const T* x = static_cast<const T*>(R.x) + R.at(r, R.s0, R.s1);
    GT* g = static_cast<GT*>(G.g) + R.at(r, G.s0, G.s1);
    if (!R.counts(r)) {
      row_zero<T, NT>(x, g, R.cols, tid, INT64_MAX);
      if (tid == 0) {
        logp[r] = 0.0f;
        put(terms, r, 0.0f, 0.0f, 0.0f);
      }
      continue;
    }
    const int64_t y = R.tokens[r];
    const float raw_y = tid == 0 ? to_f32(x[y]) : 0.0f;
    const MaxSum a = row_stats<T, NT>(x, R.cols, R.c, tid, sh);
    float coef = 0.0f;
    if (tid == 0) {
      const double lp = token_logp(raw_y, a, R.mul);
      const Token t = policy_token(P, r, lp);
      logp[r] = (float)lp;
      put(terms, r, t.loss, t.kl, t.clipped ? 1.0f : 0.0f);
      coef = (float)((double)t.coef / denom) * gain;
      if (NT > 32) coef_sh = coef;
    }
    if (NT > 32) {
      __syncthreads();
      coef = coef_sh;
      __syncthreads();  // coef_sh and sh are free again
    } else {
      coef = __shfl_sync(0xffffffffu, coef, 0);
    }
    if (coef == 0.0f)
      row_zero<T, NT>(x, g, R.cols, tid, INT64_MAX);
    else
      row_grad<T, NT>(x, g, R.cols, R.c, row_off(a.m), coef * (1.0f / a.s), coef, y, tid, INT64_MAX);
  }
}

// Fixed-order sum over a CTA of 1024 threads.
ECO_DEV double cta_sum(double v, double* sh) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0;
  for (int w = 0; w < (int)blockDim.x / 32; ++w) v += sh[w];
  __syncthreads();
  return v;
}

// loss, kl and clip fraction from the rows' terms (one CTA, fixed order, sums in double).
__global__ void __launch_bounds__(1024) policy_finish_kernel(const __grid_constant__ Rows R, const Terms terms,
                                                              double denom, float* out) {
  __shared__ double sh[32];
  __shared__ int counts_sh[32];
  const double n = policy_denom(R, denom, counts_sh);
  double a = 0.0, b = 0.0, d = 0.0;
  for (int64_t r = threadIdx.x; r < R.rows; r += blockDim.x) {
    a += terms.loss[r];
    b += terms.kl[r];
    d += terms.clip[r];
  }
  a = cta_sum(a, sh);
  b = cta_sum(b, sh);
  d = cta_sum(d, sh);
  if (threadIdx.x == 0) {
    out[0] = (float)(a / n);
    out[1] = (float)(b / n);
    out[2] = (float)(d / n);
  }
}

// The policy loss from log-probabilities: terms and coefficients (one CTA).
__global__ void __launch_bounds__(1024) policy_tokens_kernel(const __grid_constant__ Rows R,
                                                              const __grid_constant__ Policy P, const double* lp64,
                                                              float* coef, float* out) {
  __shared__ double sh[32];
  __shared__ int counts_sh[32];
  const double n = policy_denom(R, P.denom, counts_sh);
  double a = 0.0, b = 0.0, d = 0.0;
  for (int64_t r = threadIdx.x; r < R.rows; r += blockDim.x) {
    float k = 0.0f;
    if (R.counts(r)) {
      const Token t = policy_token(P, r, lp64[r]);
      a += t.loss;
      b += t.kl;
      d += t.clipped ? 1.0 : 0.0;
      k = (float)((double)t.coef / n);
    }
    coef[r] = k;
  }
  a = cta_sum(a, sh);
  b = cta_sum(b, sh);
  d = cta_sum(d, sh);
  if (threadIdx.x == 0) {
    out[0] = (float)(a / n);
    out[1] = (float)(b / n);
    out[2] = (float)(d / n);
  }
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
  __shared__ double sh[32];
  const int64_t p = blockIdx.x;
  int64_t lo[2], hi[2];
  double ratio[2], per[2];
  for (int s = 0; s < 2; ++s) {
    const int64_t q = p + s * P.pairs;
    int64_t b = R.cu ? (int64_t)R.cu[q] : q * P.seq_len, e = R.cu ? (int64_t)R.cu[q + 1] : (q + 1) * P.seq_len;
    b = b < 0 ? 0 : (b > R.rows ? R.rows : b);
    e = e < b ? b : (e > R.rows ? R.rows : e);
    double v = 0.0, n = 0.0;
    for (int64_t r = b + threadIdx.x; r < e; r += blockDim.x)
      if (R.counts(r)) {
        v += lp64[r] - (double)P.ref[r];
        n += 1.0;
      }
    v = cta_sum(v, sh);
    n = cta_sum(n, sh);
    lo[s] = b;
    hi[s] = e;
    per[s] = P.average && n > 0.0 ? 1.0 / n : 1.0;
    ratio[s] = v * per[s];
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
  for (int s = 0; s < 2; ++s) {
    const float k = (float)((s ? -slope : slope) * per[s] / P.denom);
    for (int64_t r = lo[s] + threadIdx.x; r < hi[s]; r += blockDim.x)
      if (R.counts(r)) coef[r] = k;
  }
}

__global__ void __launch_bounds__(256) pair_finish_kernel(const double* pair_loss, int64_t pairs, double denom,
                                                           float* out) {
  __shared__ double sh[32];
  double a = 0.0;
  for (int64_t p = threadIdx.x; p < pairs; p += blockDim.x) a += pair_loss[p];
  a = cta_sum(a, sh);
  if (threadIdx.x == 0) out[0] = (float)(a / denom);
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
  R.c = (float)(L.mul * 1.4426950408889634);
  R.tokens = tokens;
  R.mask = mask;
  R.cu = cu;
  R.nseq = (int)nseq;
  return R;
}

int esize(int type) { return type == ECO_F32 ? 4 : type == ECO_I8 ? 1 : 2; }

int check_logits(const eco_logits_t* L, const int64_t* tokens, const char* who) {
  ECO_REQUIRE(L && L->n0 >= 0 && L->n1 >= 0 && L->cols > 0, ECO_ERR_ARG, "%s: bad shape", who);
  ECO_REQUIRE(L->type >= ECO_F32 && L->type <= ECO_I8, ECO_ERR_ARG, "%s: unknown logits type %d", who, L->type);
  ECO_REQUIRE(L->n0 == 0 || L->n1 == 0 || (L->x && tokens), ECO_ERR_ARG, "%s: null logits or tokens", who);
  ECO_REQUIRE(std::isfinite(L->mul) && L->mul > 0.0, ECO_ERR_ARG, "%s: the logits' factor must be positive", who);
  ECO_REQUIRE(L->s0 >= 0 && L->s1 >= 0, ECO_ERR_ARG, "%s: negative strides", who);
  ECO_REQUIRE(reinterpret_cast<uintptr_t>(L->x) % (uintptr_t)esize(L->type) == 0, ECO_ERR_MISALIGNED,
              "%s: logits are not aligned to their type", who);
  ECO_REQUIRE(L->n1 == 0 || L->n0 <= INT32_MAX / L->n1, ECO_ERR_ARG, "%s: 2^31 rows or more", who);
  ECO_REQUIRE(L->cols <= (int64_t)1 << 28, ECO_ERR_ARG, "%s: more than 2^28 columns", who);
  return ECO_OK;
}

// A gradient row starts at the logits row's address modulo 16 bytes (so 16-byte vectors of
// both hold the same elements), and on 16 bytes for int8 logits.
int check_grad(const eco_logits_t& L, const eco_grad_t* G, const char* who) {
  ECO_REQUIRE(G && G->g && G->s0 >= 0 && G->s1 >= 0 && (L.n1 <= 1 || G->s1 >= L.cols) &&
                  (L.n0 <= 1 || G->s0 >= L.cols),
              ECO_ERR_ARG, "%s: bad gradient layout", who);
  const int64_t es = esize(L.type);
  const int64_t base = reinterpret_cast<uintptr_t>(G->g);
  bool ok;
  if (L.type == ECO_I8)
    ok = base % 16 == 0 && (L.n0 <= 1 || G->s0 % 4 == 0) && (L.n1 <= 1 || G->s1 % 4 == 0);
  else
    ok = (base - (int64_t) reinterpret_cast<uintptr_t>(L.x)) % 16 == 0 &&
         (L.n0 <= 1 || (G->s0 - L.s0) * es % 16 == 0) && (L.n1 <= 1 || (G->s1 - L.s1) * es % 16 == 0);
  ECO_REQUIRE(ok, ECO_ERR_MISALIGNED, "%s: gradient rows must start like the logits rows modulo 16 bytes", who);
  return ECO_OK;
}

// Threads per row: a warp up to 1024 columns (no barrier; eight rows per CTA), a CTA beyond.
int row_threads(int64_t cols) { return cols <= 1024 ? 32 : cols <= 8192 ? 128 : 512; }

template <typename F>
int by_type(int type, F f) {
  switch (type) {
    case ECO_F32: return f((float*)nullptr);
    case ECO_BF16: return f((__nv_bfloat16*)nullptr);
    case ECO_F16: return f((__half*)nullptr);
    default: return f((int8_t*)nullptr);
  }
}

template <typename T, int NT>
void launch_logp(const Rows& R, float* logp, double* lp64, float2* stats, float* coef0, cudaStream_t s) {
  constexpr int threads = NT == 32 ? 256 : NT;
  const int64_t grid = std::min<int64_t>((R.rows + threads / NT - 1) / (threads / NT), 1 << 20);
  token_logp_kernel<T, NT><<<(unsigned)grid, threads, 0, s>>>(R, logp, lp64, stats, coef0);
}

template <typename T, int NT>
void launch_policy(const Rows& R, const Policy& P, float gain, float* logp, const Terms& t, const Grad& G,
                   cudaStream_t s) {
  constexpr int threads = NT == 32 ? 256 : NT;
  const int64_t cap = (int64_t)eco_num_sms() * (1536 / threads);
  const int64_t grid = std::min<int64_t>((R.rows + threads / NT - 1) / (threads / NT), cap);
  policy_row_kernel<T, NT><<<(unsigned)grid, threads, 0, s>>>(R, P, gain, logp, t, G);
}

template <typename T>
void launch_grad(const Rows& R, const float2* stats, const float* coef, const float* scale, float gain,
                 const Grad& G, cudaStream_t s) {
  const int64_t vecs = R.cols / RowIo<T>::E + 1;
  if (R.cols <= 1024) {
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
    const int nt = row_threads(R.cols);
    if (nt == 32) launch_logp<T, 32>(R, logp, logp64, st, coef_zero, eco_stream(stream));
    else if (nt == 128) launch_logp<T, 128>(R, logp, logp64, st, coef_zero, eco_stream(stream));
    else launch_logp<T, 512>(R, logp, logp64, st, coef_zero, eco_stream(stream));
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
  by_type(logits->type, [&](auto* p) {
    using T = std::remove_pointer_t<decltype(p)>;
    const int nt = row_threads(R.cols);
    if (nt == 32) launch_policy<T, 32>(R, P, (float)gain, logp, t, G, s);
    else if (nt == 128) launch_policy<T, 128>(R, P, (float)gain, logp, t, G, s);
    else launch_policy<T, 512>(R, P, (float)gain, logp, t, G, s);
    return 0;
  });
  policy_finish_kernel<<<1, 1024, 0, s>>>(R, t, denom, out);
  return eco_launch_check("eco_policy_grad");
}

extern "C" int eco_policy_tokens(const double* logp64, const int64_t* tokens, const uint8_t* mask, int64_t rows,
                                 int64_t cols, const float* old_logp, const float* adv, const float* ref_logp,
                                 double low, double high, double kl_coef, double denom, float* coef, float* out,
                                 eco_stream_t stream) {
  ECO_REQUIRE(rows >= 0 && cols > 0 && out, ECO_ERR_ARG, "eco_policy_tokens: bad arguments");
  cudaStream_t s = eco_stream(stream);
  if (rows == 0) {
    if (cudaMemsetAsync(out, 0, 3 * sizeof(float), s) != cudaSuccess) return eco_launch_check("eco_policy_tokens");
    return ECO_OK;
  }
  Policy P;
  if (int rc = policy_of(P, old_logp, adv, ref_logp, low, high, kl_coef, denom, "eco_policy_tokens")) return rc;
  ECO_REQUIRE(logp64 && tokens && coef, ECO_ERR_ARG, "eco_policy_tokens: null pointers");
  const eco_logits_t L{nullptr, ECO_F32, 0, 1, rows, 0, 0, cols, 1.0};
  const Rows R = rows_of(L, tokens, mask, nullptr, 0);
  policy_tokens_kernel<<<1, 1024, 0, s>>>(R, P, logp64, coef, out);
  return eco_launch_check("eco_policy_tokens");
}

extern "C" int eco_preference_pairs(const double* logp64, const int64_t* tokens, const uint8_t* mask, int64_t rows,
                                    int64_t cols, const float* ref_logp, const int32_t* cu_seqlens, int64_t seq_len,
                                    int64_t pairs, int kind, double beta, double label_smoothing, int average,
                                    double denom, float* coef, float* log_ratio, float* margin, double* pair_loss,
                                    float* out, eco_stream_t stream) {
  ECO_REQUIRE(rows >= 0 && cols > 0 && pairs > 0 && pairs < (1 << 30) && seq_len >= 0 && log_ratio && margin &&
                  pair_loss && out && (rows == 0 || (logp64 && tokens && ref_logp && coef)),
              ECO_ERR_ARG, "eco_preference_pairs: bad arguments");
  ECO_REQUIRE(cu_seqlens || rows / 2 / pairs >= seq_len, ECO_ERR_ARG, "eco_preference_pairs: more sequences than rows");
  ECO_REQUIRE(kind >= ECO_PREFERENCE_SIGMOID && kind <= ECO_PREFERENCE_IPO, ECO_ERR_ARG,
              "eco_preference_pairs: unknown kind %d", kind);
  ECO_REQUIRE(std::isfinite(beta) && beta > 0.0 && label_smoothing >= 0.0 && label_smoothing <= 1.0 && denom > 0.0,
              ECO_ERR_ARG, "eco_preference_pairs: bad beta, smoothing or denominator");
  const eco_logits_t L{nullptr, ECO_F32, 0, 1, rows, 0, 0, cols, 1.0};
  const Rows R = rows_of(L, tokens, mask, cu_seqlens, 2 * pairs);
  const Pairs P{ref_logp, seq_len, pairs, beta, label_smoothing, denom, kind, average != 0};
  cudaStream_t s = eco_stream(stream);
  pair_kernel<<<(unsigned)pairs, 256, 0, s>>>(R, P, logp64, coef, log_ratio, margin, pair_loss);
  pair_finish_kernel<<<1, 256, 0, s>>>(pair_loss, pairs, denom, out);
  return eco_launch_check("eco_preference_pairs");
}
