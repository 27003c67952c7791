// Log probability of a given token per row of logits, the row's entropy and its largest entries; and the gradient.
//
//   m = max x,  S = sum exp(x - m),  logp = (x_y - m) - log S,  H = log S - sum p (x - m),  p = exp(x - m) / S
//   d x = g_logp (1[y] - p) - g_H p (log p + H)
//
// Both passes stream the row once with 16-byte loads and are bound by DRAM.  Forward: a block per row, eight loads in flight
// per thread, running maximum and sums per thread (fp32; a thread adds V / 256 terms, the rest is a tree), so nothing of the
// row is kept.  Differences to the maximum are formed before they are scaled: a row whose entries all are the type's lowest
// value is uniform, as it should be.
// Alternatives: every eighth thread group's maximum is an entry of the row, so the top-th largest of those 32 maxima bounds
// the top-th largest entry from below; only threads whose own maximum reaches the bound look at their part of the row again
// (from L2), and what reaches the bound, a few entries more than `top`, is ranked by (value, lower index first).
// A row has no target where its token is negative: logp = 0, no gradient through it.  A token beyond the vocabulary gives NaN.
#include <cuda_fp16.h>

#include "common.cuh"

namespace {

constexpr int NT = 256, U = 8, GROUPS = 32, MAX_TOP = 32, CAP = 1024;
constexpr float L2E = 1.4426950408889634f;
// exp of anything below this is zero in fp32; keeps 0 x (-inf) out of the sums
constexpr float LOWEST = -200.f;

// one exponential on the special-function unit; results below 2^-126 are zero
__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

template <typename T>
struct Vec;   // 16 bytes of a row
template <>
struct Vec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void get(const uint4& u, float (&f)[4]) {
    f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y); f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
  }
  static __device__ __forceinline__ uint4 put(const float (&f)[4]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
  static __device__ __forceinline__ float one(float v) { return v; }
  static __device__ __forceinline__ float from(float v) { return v; }
};
template <>
struct Vec<bf16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void get(const uint4& u, float (&f)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ uint4 put(const float (&f)[8]) {
    return make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
  }
  static __device__ __forceinline__ float one(bf16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ bf16 from(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct Vec<__half> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void get(const uint4& u, float (&f)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = v.x;
      f[2 * i + 1] = v.y;
    }
  }
  static __device__ __forceinline__ uint4 put(const float (&f)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 v = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  static __device__ __forceinline__ float one(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half from(float v) { return __float2half_rn(v); }
};

// a row as [head: up to the first 16-byte boundary) [body: vectors) [tail)
struct Cut {
  int head, nvec, tail0;
};
template <typename T>
__device__ __forceinline__ Cut cut_row(const T* x, int V) {
  const int mis = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const int head = min(V, mis ? Vec<T>::N - mis : 0);
  const int nvec = (V - head) / Vec<T>::N;
  return {head, nvec, head + nvec * Vec<T>::N};
}

// running maximum, sum of exp(x - m) and sum of exp(x - m) (x - m)
struct Run {
  float m, s, e;
  __device__ __forceinline__ void raise(float top) {          // move the reference to `top` > m
    const float d = m - top;                                  // -inf the first time
    const float f = ex2(d * L2E);
    e = f * fmaf(fmaxf(d, LOWEST), s, e);
    s *= f;
    m = top;
  }
  __device__ __forceinline__ void add(float x) {
    const float d = x - m, p = ex2(d * L2E);
    s += p;
    e = fmaf(p, fmaxf(d, LOWEST), e);
  }
  __device__ __forceinline__ void join(float m2, float s2, float e2) {
    const float top = fmaxf(m, m2);
    if (top == -INFINITY) return;
    const float d1 = m - top, d2 = m2 - top;
    const float f1 = ex2(d1 * L2E), f2 = ex2(d2 * L2E);
    e = f1 * fmaf(fmaxf(d1, LOWEST), s, e) + f2 * fmaf(fmaxf(d2, LOWEST), s2, e2);
    s = f1 * s + f2 * s2;
    m = top;
  }
};

__device__ __forceinline__ bool ahead(float v, int i, float w, int j) { return v > w || (v == w && i < j); }

// the entries of this thread's part of the row, each with its index
template <typename T, typename F>
__device__ __forceinline__ void each_own(const T* x, const Cut& c, int V, F f) {
  const int t = threadIdx.x;
  if (t < c.head) f(Vec<T>::one(x[t]), t);
  const uint4* body = reinterpret_cast<const uint4*>(x + c.head);
  for (int i = t; i < c.nvec; i += NT) {
    float v[Vec<T>::N];
    Vec<T>::get(__ldg(body + i), v);
#pragma unroll
    for (int k = 0; k < Vec<T>::N; ++k) f(v[k], c.head + i * Vec<T>::N + k);
  }
  if (c.tail0 + t < V) f(Vec<T>::one(x[c.tail0 + t]), c.tail0 + t);
}

template <typename T, bool TOP>
__global__ void __launch_bounds__(NT) logprob_fwd_kernel(const T* __restrict__ logits, long long rs,
                                                         const long long* __restrict__ tokens, int V, int top,
                                                         float* __restrict__ logp, float* __restrict__ entropy,
                                                         float2* __restrict__ stats, float* __restrict__ top_logp,
                                                         long long* __restrict__ top_ids) {
  constexpr int N = Vec<T>::N;
  const long long row = blockIdx.x;
  const T* x = logits + row * rs;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const Cut c = cut_row(x, V);
  Run r{-INFINITY, 0.f, 0.f};
  auto single = [&](float v) {
    if (v > r.m) r.raise(v);
    if (v != -INFINITY) r.add(v);                     // -inf adds nothing; NaN and +inf make the sums NaN
  };
  if (t < c.head) single(Vec<T>::one(x[t]));
  if (c.tail0 + t < V) single(Vec<T>::one(x[c.tail0 + t]));
  const uint4* body = reinterpret_cast<const uint4*>(x + c.head);
  for (int i = t; i < c.nvec; i += NT * U) {
    uint4 u[U];
#pragma unroll
    for (int k = 0; k < U; ++k)
      if (i + k * NT < c.nvec) u[k] = __ldg(body + i + k * NT);
#pragma unroll
    for (int k = 0; k < U; ++k) {
      if (i + k * NT < c.nvec) {
        float v[N];
        Vec<T>::get(u[k], v);
        float mx = v[0];
#pragma unroll
        for (int q = 1; q < N; ++q) mx = fmaxf(mx, v[q]);
        if (mx > r.m) r.raise(mx);
        if (r.m != -INFINITY) {
#pragma unroll
          for (int q = 0; q < N; ++q) r.add(v[q]);
        } else {
#pragma unroll
          for (int q = 0; q < N; ++q)
            if (v[q] != v[q]) r.s = v[q];             // nothing but -inf and NaN so far
        }
      }
    }
  }
  // ---- the block's sums ----
  __shared__ float sm[8], ss[8], se[8];
  __shared__ float s_m, s_ls;
  const float own = r.m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, r.m, o), s2 = __shfl_xor_sync(0xffffffffu, r.s, o),
                e2 = __shfl_xor_sync(0xffffffffu, r.e, o);
    // the same order of terms in both partners
    const bool low = (lane & o) == 0;
    Run z = low ? r : Run{m2, s2, e2};
    const float ms = low ? m2 : r.m, sx = low ? s2 : r.s, ex = low ? e2 : r.e;
    const bool dead = z.m == -INFINITY && ms == -INFINITY;
    z.join(ms, sx, ex);
    if (dead) z.s += sx;                              // NaN of a thread that saw nothing else
    r = z;
  }
  if (lane == 0) { sm[warp] = r.m; ss[warp] = r.s; se[warp] = r.e; }
  __shared__ float g_max[GROUPS];                     // maxima of the groups of 8 threads
  if (TOP) {
    float gm = own;
    gm = fmaxf(gm, __shfl_xor_sync(0xffffffffu, gm, 1));
    gm = fmaxf(gm, __shfl_xor_sync(0xffffffffu, gm, 2));
    gm = fmaxf(gm, __shfl_xor_sync(0xffffffffu, gm, 4));
    if ((t & 7) == 0) g_max[t >> 3] = gm;
  }
  __shared__ float s_bound;
  __shared__ int s_n;
  __syncthreads();
  if (t == 0) {
    Run z{sm[0], ss[0], se[0]};
#pragma unroll
    for (int w = 1; w < NT / 32; ++w) {
      const bool dead = z.m == -INFINITY && sm[w] == -INFINITY;
      z.join(sm[w], ss[w], se[w]);
      if (dead) z.s += ss[w];
    }
    const float ls = logf(z.s);
    const long long y = tokens[row];
    float lp = 0.f;
    if (y >= 0) lp = y < V ? (Vec<T>::one(x[y]) - z.m) - ls : NAN;
    logp[row] = lp;
    entropy[row] = ls - z.e / z.s;
    if (stats) stats[row] = make_float2(z.m, ls);
    s_m = z.m;
    s_ls = ls;
    s_n = 0;
  }
  if (!TOP) return;
  // ---- alternatives ----
  __shared__ float cv[CAP];
  __shared__ int ci[CAP];
  if (warp == 1) {                                    // the top-th largest of the group maxima
    const float v = g_max[lane];
    int rank = 0;
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) rank += ahead(g_max[i], i, v, lane);
    if (rank == top - 1) s_bound = v;
  }
  __syncthreads();
  const float bound = s_bound;
  if (!(own < bound))
    each_own(x, c, V, [&](float v, int i) {
      if (!(v < bound)) {                             // NaN goes in as well: it is ranked as the smallest
        const int at = atomicAdd(&s_n, 1);
        if (at < CAP) { cv[at] = v == v ? v : -INFINITY; ci[at] = i; }
      }
    });
  __syncthreads();
  const int n = s_n;
  if (n <= CAP) {
    for (int a = t; a < n; a += NT) {
      const float v = cv[a];
      const int i = ci[a];
      int rank = 0;
      for (int b = 0; b < n; ++b) rank += ahead(cv[b], ci[b], v, i);
      if (rank < top) {
        top_logp[row * top + rank] = (v - s_m) - s_ls;
        top_ids[row * top + rank] = i;
      }
    }
    return;
  }
  // more ties than the list holds (a constant row, a row masked down to a few entries): one entry at a time, each the
  // best behind the one before it
  float pv = INFINITY;
  int pi = -1;
  for (int k = 0; k < top; ++k) {
    float bv = -INFINITY;
    int bi = V;
    each_own(x, c, V, [&](float v, int i) {
      if (v != v) v = -INFINITY;
      if (ahead(pv, pi, v, i) && ahead(v, i, bv, bi)) { bv = v; bi = i; }
    });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float v2 = __shfl_xor_sync(0xffffffffu, bv, o);
      const int i2 = __shfl_xor_sync(0xffffffffu, bi, o);
      if (ahead(v2, i2, bv, bi)) { bv = v2; bi = i2; }
    }
    __syncthreads();
    if (lane == 0) { cv[warp] = bv; ci[warp] = bi; }
    __syncthreads();
    pv = cv[0];
    pi = ci[0];
    for (int w = 1; w < NT / 32; ++w)
      if (ahead(cv[w], ci[w], pv, pi)) { pv = cv[w]; pi = ci[w]; }
    if (t == 0) {
      top_logp[row * top + k] = (pv - s_m) - s_ls;
      top_ids[row * top + k] = pi;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(NT) logprob_bwd_kernel(const T* __restrict__ logits, long long rs,
                                                         const long long* __restrict__ tokens, int V,
                                                         const float2* __restrict__ stats, const float* __restrict__ entropy,
                                                         const float* __restrict__ g_logp, const float* __restrict__ g_ent,
                                                         T* __restrict__ dx) {
  constexpr int N = Vec<T>::N;
  const long long row = blockIdx.x;
  const T* x = logits + row * rs;
  T* out = dx + row * V;
  const int t = threadIdx.x;
  const long long y = tokens[row];
  const float2 st = stats[row];
  const float gh = g_ent ? g_ent[row] : 0.f, gl = g_logp && y >= 0 ? (y < V ? g_logp[row] : NAN) : 0.f;
  const float base = fmaf(gh, entropy[row], gl);
  const int yi = y >= 0 && y < V ? (int)y : -1;
  auto grad = [&](float v) {
    const float lp = (v - st.x) - st.y;
    return -ex2(lp * L2E) * fmaf(gh, fmaxf(lp, LOWEST), base);
  };
  // the output row is aligned like the input row or not: vectors where both are, else one by one
  const Cut c = cut_row(x, V);
  const bool same = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;
  auto single = [&](int i) {
    const float g = grad(Vec<T>::one(x[i]));
    out[i] = Vec<T>::from(i == yi ? g + gl : g);
  };
  if (t < c.head) single(t);
  if (c.tail0 + t < V) single(c.tail0 + t);
  const uint4* body = reinterpret_cast<const uint4*>(x + c.head);
  constexpr int UB = 4;
  for (int i = t; i < c.nvec; i += NT * UB) {
    uint4 u[UB];
#pragma unroll
    for (int k = 0; k < UB; ++k)
      if (i + k * NT < c.nvec) u[k] = __ldg(body + i + k * NT);
#pragma unroll
    for (int k = 0; k < UB; ++k) {
      const int j = i + k * NT;
      if (j < c.nvec) {
        float v[N];
        Vec<T>::get(u[k], v);
        const int e0 = c.head + j * N;
#pragma unroll
        for (int q = 0; q < N; ++q) {
          v[q] = grad(v[q]);
          if (e0 + q == yi) v[q] += gl;
        }
        if (same) {
          *reinterpret_cast<uint4*>(out + e0) = Vec<T>::put(v);
        } else {
#pragma unroll
          for (int q = 0; q < N; ++q) out[e0 + q] = Vec<T>::from(v[q]);
        }
      }
    }
  }
}

template <typename T>
int fwd(const void* x, long long rs, const long long* tok, long long rows, int V, int top, float* lp, float* ent, float2* st,
        float* tlp, long long* tid, cudaStream_t s) {
  if (top > 0)
    logprob_fwd_kernel<T, true><<<(unsigned)rows, NT, 0, s>>>((const T*)x, rs, tok, V, top, lp, ent, st, tlp, tid);
  else
    logprob_fwd_kernel<T, false><<<(unsigned)rows, NT, 0, s>>>((const T*)x, rs, tok, V, top, lp, ent, st, tlp, tid);
  DMB_CHECK_LAUNCH();
  return 0;
}
template <typename T>
int bwd(const void* x, long long rs, const long long* tok, long long rows, int V, const float2* st, const float* ent,
        const float* gl, const float* gh, void* dx, cudaStream_t s) {
  logprob_bwd_kernel<T><<<(unsigned)rows, NT, 0, s>>>((const T*)x, rs, tok, V, st, ent, gl, gh, (T*)dx);
  DMB_CHECK_LAUNCH();
  return 0;
}

}  // namespace

// logits [rows, V] with row stride rs (elements) and dense columns; type: 0 fp32, 1 bf16, 2 fp16; tokens int64 [rows];
// logp / entropy fp32 [rows]; stats fp32 [rows, 2] (maximum, log of the sum) or null; top_logp / top_ids [rows, top]
extern "C" int dmb_logprob_fwd(const void* x, long long rs, const long long* tokens, long long rows, int V, int type, int top,
                               float* logp, float* entropy, float* stats, float* top_logp, long long* top_ids, void* stream) {
  if (rows <= 0) return 0;
  if (V <= 0 || rows > 0x7fffffffLL || top < 0 || top > MAX_TOP || top > V) return -1;
  cudaStream_t s = (cudaStream_t)stream;
  float2* st = (float2*)stats;
  if (type == 0) return fwd<float>(x, rs, tokens, rows, V, top, logp, entropy, st, top_logp, top_ids, s);
  if (type == 1) return fwd<bf16>(x, rs, tokens, rows, V, top, logp, entropy, st, top_logp, top_ids, s);
  if (type == 2) return fwd<__half>(x, rs, tokens, rows, V, top, logp, entropy, st, top_logp, top_ids, s);
  return -1;
}
// dx [rows, V] dense; g_logp / g_entropy fp32 [rows] or null (no gradient through that output)
extern "C" int dmb_logprob_bwd(const void* x, long long rs, const long long* tokens, long long rows, int V, int type,
                               const float* stats, const float* entropy, const float* g_logp, const float* g_entropy, void* dx,
                               void* stream) {
  if (rows <= 0) return 0;
  if (V <= 0 || rows > 0x7fffffffLL) return -1;
  cudaStream_t s = (cudaStream_t)stream;
  const float2* st = (const float2*)stats;
  if (type == 0) return bwd<float>(x, rs, tokens, rows, V, st, entropy, g_logp, g_entropy, dx, s);
  if (type == 1) return bwd<bf16>(x, rs, tokens, rows, V, st, entropy, g_logp, g_entropy, dx, s);
  if (type == 2) return bwd<__half>(x, rs, tokens, rows, V, st, entropy, g_logp, g_entropy, dx, s);
  return -1;
}
