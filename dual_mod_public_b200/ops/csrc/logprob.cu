// Log probability of a given token per row of logits, the row's entropy and its largest entries; and the gradient.
//
//   m = max x,  S = sum exp(x - m),  logp = (x_y - m) - log S,  H = log S - sum p (x - m),  p = exp(x - m) / S
//   d x = g_logp (1[y] - p) - g_H p (log p + H)
//
// Both passes stream the row once with 16-byte loads and are bound by DRAM (8191 x 32000 bf16: forward 95 us, 5.5 TB/s, with the
// greedy entry 102 us, with eight alternatives 137 us; the exponentials take 60 % of the special-function unit meanwhile;
// backward 169 us, 6.2 TB/s).  -inf among a thread's entries sends its set of vectors through a scalar loop (every second entry: 307
// us).  Forward: a group of 32 to 1024 threads per row (see `fwd`), two sets of loads in flight per thread, running maximum and sums per thread
// (fp32; a thread adds its part of the row, the rest is a tree).  A block takes rows in turn and requests the next row's first
// part before it joins the sums of the last.  A row whose entries all are the type's lowest value is uniform, as it should be.
// The rows in flight may not fit L2, so reading an entry again costs a round trip to DRAM under load.  The greedy entry does
// without: a thread keeps the set of vectors that its maximum came with in shared memory (116 -> 108 us when built).
// Alternatives: the maxima of 32 parts of the row are entries of it, so the top-th largest of them bounds the top-th largest
// entry from below; only threads whose own maximum reaches the bound have their entries looked at again, and what reaches
// the bound, a few entries more than `top`, is ranked by (value, lower index first).
// A row has no target where its token is negative: logp = 0, no gradient through it.  A token beyond the vocabulary gives NaN.
#include <climits>

#include "packed.cuh"

namespace {

constexpr int MAX_TOP = 32;
constexpr float L2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
// exp of anything below this is zero in fp32; keeps 0 x (-inf) out of the sums
constexpr float LOWEST = -200.f;

using packed::ex2;

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
  static __device__ __forceinline__ float top(const uint4& u) {       // the largest, NaN aside
    return fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)), fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
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
  static __device__ __forceinline__ float top(const uint4& u) {
    auto h = [](uint32_t w) { return *reinterpret_cast<const bf162*>(&w); };
    const bf162 m = __hmax2(__hmax2(h(u.x), h(u.y)), __hmax2(h(u.z), h(u.w)));
    return fmaxf(__bfloat162float(m.x), __bfloat162float(m.y));
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
  static __device__ __forceinline__ float top(const uint4& u) {
    auto h = [](uint32_t w) { return *reinterpret_cast<const __half2*>(&w); };
    const __half2 m = __hmax2(__hmax2(h(u.x), h(u.y)), __hmax2(h(u.z), h(u.w)));
    return fmaxf(__half2float(m.x), __half2float(m.y));
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

// Running maximum m, s = sum of 2^y and e = sum of 2^y y with y = x log2(e) - ref, ref the whole number above m log2(e): the
// product and the difference are one rounding of a small value, and moving ref scales the sums by an exact power of two.
// Where |m| is above 1e9 (rows of a mask's value, infinities) differences are formed first and ref is not used.  Up to there m log2(e)
// lies within 64 of ref, half of what fp32 values of that size are apart: the maximum's own 2^y is at most 2^65.  Above, distinct
// values differ by at least 64, so sums relative to a smaller maximum count for nothing and are dropped.
struct Run {
  float m, ref, s, e;
  static __device__ __forceinline__ bool plain(float v) { return fabsf(v) <= 1e9f; }
  __device__ __forceinline__ void raise(float top) {          // `top` > m
    if (plain(m) && plain(top)) {
      const float r = ceilf(top * L2E), k = ref - r, f = ex2(k);
      e = f * fmaf(k, s, e);
      s *= f;
      ref = r;
    } else {                                                  // nothing so far, or nothing that counts beside `top` (NaN stays)
      s *= 0.f;
      e *= 0.f;
      ref = plain(top) ? ceilf(top * L2E) : 0.f;
    }
    m = top;
  }
  __device__ __forceinline__ void one(float v) {
    if (v > m) raise(v);
    if (v == -INFINITY) return;                               // adds nothing, also where m is -inf
    const float y = plain(m) ? fmaf(v, L2E, -ref) : (v - m) * L2E, p = ex2(y);
    s += p;
    e = fmaf(p, fmaxf(y, LOWEST), e);
  }
  // K vectors at once; `live` of them count.  Returns whether the maximum moved.
  template <typename T, int K>
  __device__ __forceinline__ bool many(const uint4 (&u)[K], int live) {
    constexpr int N = Vec<T>::N;
    float top = -INFINITY;
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (k < live) top = fmaxf(top, Vec<T>::top(u[k]));
    const bool up = top > m;
    if (up) raise(top);
    if (plain(m)) {
      // pairs: a packed instruction takes as long as two, but one place in the issue queue
      using namespace packed;
      const f32x2 scale = pair(L2E, L2E), off = pair(-ref, -ref);
      f32x2 ss = pair(0.f, 0.f), ee = ss;
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (k < live) {
          float v[N];
          Vec<T>::get(u[k], v);
#pragma unroll
          for (int i = 0; i < N; i += 2) {
            const f32x2 y = fma2(pair(v[i], v[i + 1]), scale, off);
            float y0, y1;
            split(y, y0, y1);
            const f32x2 q = pair(ex2(y0), ex2(y1));
            ss = add2(ss, q);
            ee = fma2(q, y, ee);
          }
        }
      float s0, s1, e0, e1;
      split(ss, s0, s1);
      split(ee, e0, e1);
      if (e0 + e1 == e0 + e1) {
        s += s0 + s1;
        e += e0 + e1;
        return up;
      }
    }
#pragma unroll 1
    for (int k = 0; k < K; ++k) {                             // -inf among them (0 x inf above), NaN, huge values: one by one
      uint4 w = u[0];
#pragma unroll
      for (int q = 1; q < K; ++q)
        if (q == k) w = u[q];
      float v[N];
      Vec<T>::get(w, v);
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (k < live) one(v[i]);
    }
    return up;
  }
  // the sums relative to m itself, e in natural units
  __device__ __forceinline__ void finish() {
    const float t = plain(m) ? fmaf(m, L2E, -ref) : 0.f, f = 1.f / ex2(t);     // the maximum's own term becomes 1
    e = f * LN2 * fmaf(-t, s, e);
    s *= f;
  }
};

__device__ __forceinline__ bool ahead(float v, int i, float w, int j) { return v > w || (v == w && i < j); }

__device__ __forceinline__ uint4 load_stream(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// A group of NT threads per row; a block is a group, or eight warps with a row each.
template <int NT>
struct Group {
  static constexpr int BLOCK = NT == 32 ? 256 : NT, ROWS = BLOCK / NT, WARPS = NT / 32;
  static constexpr int BLOCKS = 1024 / BLOCK;                 // on an SM: 64 registers a thread
  static constexpr int CAP = NT == 32 ? 96 : 1024;            // candidates that a list holds
  static __device__ __forceinline__ void sync() {
    if (NT == 32) __syncwarp(); else __syncthreads();
  }
};
enum Top { NONE, GREEDY, RANKED };
constexpr int AHEAD = 4;                                      // vectors of a set of loads
template <int NT, Top TOP>
struct Shared {                                               // of one group
  static constexpr int CAP = TOP == RANKED ? Group<NT>::CAP : 1;
  float m[Group<NT>::WARPS], s[Group<NT>::WARPS], e[Group<NT>::WARPS], part[32];
  int n, first[Group<NT>::WARPS];
  float cv[CAP];
  int ci[CAP];
  uint4 kept[AHEAD][TOP == GREEDY ? NT : 1];                  // the vectors that a thread's maximum came with, the first's place
  int kept_i[TOP == GREEDY ? NT : 1];
};

template <int NT, typename T, Top TOP>
__global__ void __launch_bounds__(Group<NT>::BLOCK, Group<NT>::BLOCKS)
logprob_fwd_kernel(const T* __restrict__ logits, long long rs, const long long* __restrict__ tokens, int rows, int V, int top,
                   float* __restrict__ logp, float* __restrict__ entropy, float2* __restrict__ stats,
                   float* __restrict__ top_logp, long long* __restrict__ top_ids) {
  using G = Group<NT>;
  constexpr int N = Vec<T>::N, K = AHEAD, CAP = Shared<NT, TOP>::CAP;
  __shared__ Shared<NT, TOP> shared[G::ROWS];
  Shared<NT, TOP>& sh = shared[threadIdx.x / NT];
  const int t = threadIdx.x % NT, lane = t & 31, warp = t >> 5;
  const long long step = (long long)gridDim.x * G::ROWS;
  long long row = (long long)blockIdx.x * G::ROWS + threadIdx.x / NT;
  if (row >= rows) return;                                    // a whole group leaves
  const T* x = logits + row * rs;
  Cut c = cut_row(x, V);
  // two sets of K vectors are in flight: vectors t + NT k of the body, k = 0 .. K - 1 and K .. 2 K - 1, then on
  uint4 a[K], b[K];
  auto fetch = [&](uint4 (&u)[K], const T* xr, const Cut& cr, int i) {
    const uint4* body = reinterpret_cast<const uint4*>(xr + cr.head);
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (i + k * NT < cr.nvec) u[k] = load_stream(body + i + k * NT);
  };
  // everything that a row's sums wait for is requested a row ahead
  T edge0 = T(), edge1 = T();                                 // this thread's entry before and behind the vectors
  long long y = 0;
  auto fetch_first = [&](const T* xr, const Cut& cr, long long r) {
    fetch(a, xr, cr, t);
    fetch(b, xr, cr, t + K * NT);
    if (t < cr.head) edge0 = xr[t];
    if (cr.tail0 + t < V) edge1 = xr[cr.tail0 + t];
    y = tokens[r];
  };
  fetch_first(x, c, row);
  for (;;) {
    Run r{-INFINITY, 0.f, 0.f, 0.f};
    const long long target = y;
    auto take = [&](const uint4 (&u)[K], int i) {
      if (r.template many<T, K>(u, min(K, (c.nvec - i + NT - 1) / NT)) && TOP == GREEDY) {
        sh.kept_i[t] = i;
#pragma unroll
        for (int k = 0; k < K; ++k) sh.kept[k][t] = u[k];
      }
    };
    for (int i = t; i < c.nvec; i += 2 * K * NT) {
      take(a, i);
      fetch(a, x, c, i + 2 * K * NT);
      if (i + K * NT < c.nvec) take(b, i + K * NT);
      fetch(b, x, c, i + 3 * K * NT);
    }
    const float best = r.m, head = t < c.head ? Vec<T>::one(edge0) : NAN, tail = c.tail0 + t < V ? Vec<T>::one(edge1) : NAN;
    if (t < c.head) r.one(head);
    if (c.tail0 + t < V) r.one(tail);
    // the next row's first vectors travel while this row's sums are joined
    const long long next = row + step;
    const T* xn = logits + next * rs;
    Cut cn = c;
    if (next < rows) {
      cn = cut_row(xn, V);
      fetch_first(xn, cn, next);
    }
    float xy = 0.f;
    if (t == 0 && target >= 0 && target < V) xy = Vec<T>::one(x[target]);
    // ---- the row's sums: within the warp, then across warps ----
    const float own = r.m;
    if (TOP == RANKED) {                                      // maxima of the groups of NT / 32 threads
      float part = own;
#pragma unroll
      for (int o = 1; o < NT / 32; o <<= 1) part = fmaxf(part, __shfl_xor_sync(0xffffffffu, part, o));
      if (t % (NT / 32) == 0) sh.part[t / (NT / 32)] = part;
    }
    auto join = [&](float& m, float& s, float& e, int width) {
      float top_m = m;
#pragma unroll
      for (int o = width / 2; o > 0; o >>= 1) top_m = fmaxf(top_m, __shfl_xor_sync(0xffffffffu, top_m, o));
      if (top_m != -INFINITY) {
        const float d = m - top_m, f = ex2(d * L2E);
        e = f * fmaf(fmaxf(d, LOWEST), s, e);
        s *= f;
      }
      m = top_m;
#pragma unroll
      for (int o = width / 2; o > 0; o >>= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, o);
        e += __shfl_xor_sync(0xffffffffu, e, o);
      }
    };
    r.finish();
    join(r.m, r.s, r.e, 32);
    if (G::WARPS > 1) {
      if (lane == 0) { sh.m[warp] = r.m; sh.s[warp] = r.s; sh.e[warp] = r.e; }
      if (t == 0) sh.n = 0;
      G::sync();
      r = Run{sh.m[lane % G::WARPS], 0.f, sh.s[lane % G::WARPS], sh.e[lane % G::WARPS]};
      join(r.m, r.s, r.e, G::WARPS);                          // every warp for itself, the same bits in all
    } else {
      if (t == 0) sh.n = 0;
      G::sync();
    }
    // The sum has a term of one and its other terms are positive, those of e negative: roundings do not carry over that, so a log
    // probability is at most zero and an entropy at least (a NaN stays, and so do the zeros of a row of nothing but -inf).
    if (r.s < 1.f && r.m > -INFINITY) r.s = 1.f;
    if (r.e > 0.f) r.e = 0.f;
    const float ls = logf(r.s);
    if (t == 0) {
      logp[row] = target < 0 ? 0.f : target < V ? (xy - r.m) - ls : NAN;
      entropy[row] = ls - r.e / r.s;
      if (stats) stats[row] = make_float2(r.m, ls);
    }
    // ---- the largest entry alone: its first place ----
    if (TOP == GREEDY) {
      int at = V;
      if (r.m == -INFINITY) at = 0;                           // nothing but -inf and NaN
      else if (head == r.m) at = t;
      else if (best == r.m) {
        const int i0 = sh.kept_i[t];
#pragma unroll
        for (int k = K - 1; k >= 0; --k)
          if (i0 + k * NT < c.nvec) {
            float v[N];
            Vec<T>::get(sh.kept[k][t], v);
#pragma unroll
            for (int i = N - 1; i >= 0; --i)
              if (v[i] == r.m) at = c.head + (i0 + k * NT) * N + i;
          }
      } else if (tail == r.m) at = c.tail0 + t;
      at = __reduce_min_sync(0xffffffffu, at);
      if (G::WARPS > 1) {
        if (lane == 0) sh.first[warp] = at;
        G::sync();
        at = __reduce_min_sync(0xffffffffu, sh.first[lane % G::WARPS]);
      }
      if (t == 0) {
        top_logp[row] = (r.m - r.m) - ls;
        top_ids[row] = at;
      }
    }
    // ---- alternatives ----
    if (TOP == RANKED) {
      float bound = r.m;
      if (top > 1) {
        const float v0 = sh.part[lane];                       // every warp ranks the 32 maxima
        int rank0 = 0;
#pragma unroll
        for (int i = 0; i < 32; ++i) rank0 += ahead(__shfl_sync(0xffffffffu, v0, i), i, v0, lane);
        bound = __shfl_sync(0xffffffffu, v0, __ffs(__ballot_sync(0xffffffffu, rank0 == top - 1)) - 1);
      }
      auto each_own = [&](auto f) {                           // this thread's entries, each with its index
        if (t < c.head) f(Vec<T>::one(x[t]), t);
        const uint4* body = reinterpret_cast<const uint4*>(x + c.head);
#pragma unroll 4
        for (int i = t; i < c.nvec; i += NT) {
          float v[N];
          Vec<T>::get(__ldg(body + i), v);
#pragma unroll
          for (int k = 0; k < N; ++k) f(v[k], c.head + i * N + k);
        }
        if (c.tail0 + t < V) f(Vec<T>::one(x[c.tail0 + t]), c.tail0 + t);
      };
      auto offer = [&](float v, int i) {
        if (!(v < bound)) {                                   // NaN goes in as well: it is ranked as the smallest
          const int at = atomicAdd(&sh.n, 1);                 // the list's order does not matter: it is ranked
          if (at < CAP) { sh.cv[at] = v == v ? v : -INFINITY; sh.ci[at] = i; }
        }
      };
      if (NT == 32) {
        if (!(own < bound)) each_own(offer);
      } else {
        // the warp looks at such threads' entries together, LOOK stretches of 32 vectors in flight (8191 x 32000 bf16, top 8:
        // 1: 152, 2: 149, 4: 160 us)
        constexpr int LOOK = 2;
        const uint4* body = reinterpret_cast<const uint4*>(x + c.head);
        unsigned left = __ballot_sync(0xffffffffu, !(own < bound));
        int from = 0;                                         // next vector of the thread that is looked at, in its own count
        while (left) {
          uint4 u[LOOK];
          int at[LOOK];
#pragma unroll
          for (int k = 0; k < LOOK; ++k) {
            const int tt = warp * 32 + __ffs(left) - 1;
            at[k] = left ? tt + NT * (from + lane) : c.nvec;
            if (at[k] < c.nvec) u[k] = __ldg(body + at[k]);
            from += 32;
            if (from * NT >= c.nvec) { from = 0; left &= left - 1; }
          }
#pragma unroll
          for (int k = 0; k < LOOK; ++k)
            if (at[k] < c.nvec && !(Vec<T>::top(u[k]) < bound)) {        // all NaN: true
              float v[N];
              Vec<T>::get(u[k], v);
#pragma unroll
              for (int i = 0; i < N; ++i) offer(v[i], c.head + at[k] * N + i);
            }
        }
        if (!(own < bound)) {
          if (t < c.head) offer(Vec<T>::one(x[t]), t);
          if (c.tail0 + t < V) offer(Vec<T>::one(x[c.tail0 + t]), c.tail0 + t);
        }
      }
      G::sync();
      const int n = sh.n;
      if (n <= CAP) {
        for (int q = t; q < n; q += NT) {
          const float v = sh.cv[q];
          const int i = sh.ci[q];
          int rank = 0;
          for (int w = 0; w < n; ++w) rank += ahead(sh.cv[w], sh.ci[w], v, i);
          if (rank < top) {
            top_logp[row * top + rank] = (v - r.m) - ls;
            top_ids[row * top + rank] = i;
          }
        }
      } else {
        // more ties than the list holds (a constant row, a row masked down to a few entries): one entry at a time, each the
        // best behind the one before it
        float pv = INFINITY;
        int pi = -1;
        for (int k = 0; k < top; ++k) {
          float bv = -INFINITY;
          int bi = V;
          each_own([&](float v, int i) {
            if (v != v) v = -INFINITY;
            if (ahead(pv, pi, v, i) && ahead(v, i, bv, bi)) { bv = v; bi = i; }
          });
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) {
            const float v2 = __shfl_xor_sync(0xffffffffu, bv, o);
            const int i2 = __shfl_xor_sync(0xffffffffu, bi, o);
            if (ahead(v2, i2, bv, bi)) { bv = v2; bi = i2; }
          }
          G::sync();
          if (lane == 0) { sh.cv[warp] = bv; sh.ci[warp] = bi; }
          G::sync();
          pv = sh.cv[0];
          pi = sh.ci[0];
          for (int w = 1; w < G::WARPS; ++w)
            if (ahead(sh.cv[w], sh.ci[w], pv, pi)) { pv = sh.cv[w]; pi = sh.ci[w]; }
          if (t == 0) {
            top_logp[row * top + k] = (pv - r.m) - ls;
            top_ids[row * top + k] = pi;
          }
        }
      }
    }
    if (next >= rows) return;
    G::sync();                                                // the shared words are free
    row = next;
    x = xn;
    c = cn;
  }
}

template <int NT, typename T>
__global__ void __launch_bounds__(Group<NT>::BLOCK) logprob_bwd_kernel(const T* __restrict__ logits, long long rs,
                                                         const long long* __restrict__ tokens, int rows, int V,
                                                         const float2* __restrict__ stats, const float* __restrict__ entropy,
                                                         const float* __restrict__ g_logp, const float* __restrict__ g_ent,
                                                         T* __restrict__ dx, int part) {
  constexpr int N = Vec<T>::N;
  const long long row = (long long)blockIdx.x * Group<NT>::ROWS + threadIdx.x / NT;
  if (row >= rows) return;
  const T* x = logits + row * rs;
  T* out = dx + row * V;
  const int t = threadIdx.x % NT;
  const long long y = tokens[row];
  const float2 st = stats[row];
  const float gh = g_ent ? g_ent[row] : 0.f, gl = g_logp && y >= 0 ? (y < V ? g_logp[row] : NAN) : 0.f;
  const float base = fmaf(gh, entropy[row], gl);
  const int yi = y >= 0 && y < V ? (int)y : -1;
  const bool none = y < 0 && gh == 0.f;                       // no gradient reaches the row: zero also where its p is NaN
  auto grad = [&](float v) {
    if (none) return 0.f;
    const float lp = (v - st.x) - st.y;
    return -ex2(lp * L2E) * fmaf(gh, fmaxf(lp, LOWEST), base);
  };
  // the output row is aligned like the input row or not: vectors where both are, else one by one
  const Cut c = cut_row(x, V);
  const int v_begin = blockIdx.y * part, v_end = min(c.nvec, v_begin + part);        // this block's vectors
  const bool same = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;
  auto single = [&](int i) {
    const float g = grad(Vec<T>::one(x[i]));
    out[i] = Vec<T>::from(i == yi ? g + gl : g);
  };
  if (blockIdx.y == 0) {
    if (t < c.head) single(t);
    if (c.tail0 + t < V) single(c.tail0 + t);
  }
  const uint4* body = reinterpret_cast<const uint4*>(x + c.head);
  constexpr int UB = 4;
  for (int i = v_begin + t; i < v_end; i += NT * UB) {
    uint4 u[UB];
#pragma unroll
    for (int k = 0; k < UB; ++k)
      if (i + k * NT < v_end) u[k] = load_stream(body + i + k * NT);
#pragma unroll
    for (int k = 0; k < UB; ++k) {
      const int j = i + k * NT;
      if (j < v_end) {
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

constexpr int SMS = 148;

template <int NT, typename T>
int fwd_nt(const T* x, long long rs, const long long* tok, int rows, int V, int top, float* lp, float* ent, float2* st, float* tlp,
           long long* tid, cudaStream_t s) {
  using G = Group<NT>;
  // as many blocks as are resident (sharing the rows out evenly over fewer blocks was slower: 108 against 102 us)
  const int grid = min((rows - 1) / G::ROWS + 1, SMS * G::BLOCKS);
  // one entry: from the sets of vectors that the threads keep in shared memory (64 bytes each, so not with 1024 threads)
  constexpr Top ONE = NT < 1024 ? GREEDY : RANKED;
  auto kern = top == 0 ? logprob_fwd_kernel<NT, T, NONE> : top == 1 ? logprob_fwd_kernel<NT, T, ONE> : logprob_fwd_kernel<NT, T, RANKED>;
  kern<<<grid, G::BLOCK, 0, s>>>(x, rs, tok, rows, V, top, lp, ent, st, tlp, tid);
  DMB_CHECK_LAUNCH();
  return 0;
}
// Threads per row.  Few threads: little to join per row; many: a row alone goes fast.  A warp where a row is short (16384 x 259:
// 27 us against 420 with 256 threads); 1024 where every row has an SM to itself; between them as few as keep two rounds of
// rows (8191 x 32000 bf16: 64 threads 102, 128 108, 256 113 us; 1021 x 50257 fp32: 128 61, 256 53 us).  Ranking alternatives
// wants more of them (8191 x 32000, top 8: 64 176, 128 152, 256 172 us before its loads went two at a time).
template <typename T>
int fwd(const void* xv, long long rs, const long long* tok, int rows, int V, int top, float* lp, float* ent, float2* st,
        float* tlp, long long* tid, cudaStream_t s) {
  const T* x = (const T*)xv;
  if (V <= 2048) return fwd_nt<32>(x, rs, tok, rows, V, top, lp, ent, st, tlp, tid, s);
  if (rows <= SMS) return fwd_nt<1024>(x, rs, tok, rows, V, top, lp, ent, st, tlp, tid, s);
  if (top <= 1 && rows >= 2 * 16 * SMS) return fwd_nt<64>(x, rs, tok, rows, V, top, lp, ent, st, tlp, tid, s);
  if (rows >= 2 * 8 * SMS) return fwd_nt<128>(x, rs, tok, rows, V, top, lp, ent, st, tlp, tid, s);
  return fwd_nt<256>(x, rs, tok, rows, V, top, lp, ent, st, tlp, tid, s);
}
template <int NT, typename T>
int bwd_nt(const T* x, long long rs, const long long* tok, int rows, int V, const float2* st, const float* ent, const float* gl,
           const float* gh, T* dx, cudaStream_t s) {
  using G = Group<NT>;
  // few rows: a row in parts of 2048 vectors (1021 x 50257 fp32: 74 against 82 us); many: whole rows (8191 x 32000 bf16: 169
  // against 178 us)
  const int nvec = V / Vec<T>::N + 1, part = rows < 4 * 8 * SMS ? max(2048, nvec / 65535 + 1) : nvec, parts = (nvec - 1) / part + 1;
  logprob_bwd_kernel<NT, T><<<dim3((rows - 1) / G::ROWS + 1, parts), G::BLOCK, 0, s>>>(x, rs, tok, rows, V, st, ent, gl, gh, dx, part);
  DMB_CHECK_LAUNCH();
  return 0;
}
template <typename T>
int bwd(const void* xv, long long rs, const long long* tok, int rows, int V, const float2* st, const float* ent,
        const float* gl, const float* gh, void* dx, cudaStream_t s) {
  const T* x = (const T*)xv;
  if (V <= 2048) return bwd_nt<32>(x, rs, tok, rows, V, st, ent, gl, gh, (T*)dx, s);
  return bwd_nt<256>(x, rs, tok, rows, V, st, ent, gl, gh, (T*)dx, s);
}

}  // namespace

// logits [rows, V] with row stride rs (elements) and dense columns; type: 0 fp32, 1 bf16, 2 fp16; tokens int64 [rows];
// logp / entropy fp32 [rows]; stats fp32 [rows, 2] (maximum, log of the sum) or null; top_logp / top_ids [rows, top]
extern "C" int dmb_logprob_fwd(const void* x, long long rs, const long long* tokens, long long rows, int V, int type, int top,
                               float* logp, float* entropy, float* stats, float* top_logp, long long* top_ids, void* stream) {
  if (rows <= 0) return 0;
  if (V <= 0 || V > INT_MAX - 4095 || rows > 0x7fffffffLL || top < 0 || top > MAX_TOP || top > V) return -1;
  cudaStream_t s = (cudaStream_t)stream;
  float2* st = (float2*)stats;
  if (type == 0) return fwd<float>(x, rs, tokens, (int)rows, V, top, logp, entropy, st, top_logp, top_ids, s);
  if (type == 1) return fwd<bf16>(x, rs, tokens, (int)rows, V, top, logp, entropy, st, top_logp, top_ids, s);
  if (type == 2) return fwd<__half>(x, rs, tokens, (int)rows, V, top, logp, entropy, st, top_logp, top_ids, s);
  return -1;
}
// dx [rows, V] dense; g_logp / g_entropy fp32 [rows] or null (no gradient through that output)
extern "C" int dmb_logprob_bwd(const void* x, long long rs, const long long* tokens, long long rows, int V, int type,
                               const float* stats, const float* entropy, const float* g_logp, const float* g_entropy, void* dx,
                               void* stream) {
  if (rows <= 0) return 0;
  if (V <= 0 || V > INT_MAX - 4095 || rows > 0x7fffffffLL) return -1;
  cudaStream_t s = (cudaStream_t)stream;
  const float2* st = (const float2*)stats;
  if (type == 0) return bwd<float>(x, rs, tokens, (int)rows, V, st, entropy, g_logp, g_entropy, dx, s);
  if (type == 1) return bwd<bf16>(x, rs, tokens, (int)rows, V, st, entropy, g_logp, g_entropy, dx, s);
  if (type == 2) return bwd<__half>(x, rs, tokens, (int)rows, V, st, entropy, g_logp, g_entropy, dx, s);
  return -1;
}
