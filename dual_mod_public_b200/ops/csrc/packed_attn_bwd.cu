// Backward of the causal attention over packed sequences (packed_attn_fwd.cu), bf16, on the 5th-generation tensor cores.
//
//   p_ij = exp(s_ij - lse_i),  delta_i = do_i . o_i,  ds_ij = p_ij (do_i . v_j - delta_i)
//   dv_j = sum_i p_ij do_i,   dk_j = scale sum_i ds_ij q_i,   dq_i = scale sum_j ds_ij k_j
//
// Two kinds of CTA in one launch, each owning what it writes, so nothing is accumulated through memory and results do not depend
// on any order:
//   dkv   a CTA per (key head, 128 keys); streams the query tiles (of all heads of the group) that see the keys.  Scores are
//         formed transposed, S^T = K Q^T and dP^T = V dO^T: a key per lane of tensor memory, so P^T and dS^T are written
//         back there as the A operands of dV += P^T dO and dK += dS^T Q
//   dq    a CTA per (query head, 128 queries); streams the key blocks: S = Q K^T, dP = dO V^T, dQ += dS K
// The price is that S and dP are formed twice (seven products of 128 x 128 x D per tile instead of five); one kernel would
// have to add dQ tiles through memory in whatever order its CTAs run.
//
// The parts of a step depend on one another: product, 500 cycles until its result is seen, exponentials, product.  So two steps
// are in work on an SM at any time, each on four math warps (a thread owns a row of the step's 128 x 128 scores, or the fragment
// of an MMA): at D = 64 in two CTAs of 256 columns of tensor memory, which also start and end independently of one another; at
// D = 128, where the accumulators fill the columns, in one CTA whose two sets of warps take the steps in turn.  One warp issues
// all products in a fixed order, one loads.  Tensor memory holds the accumulators and per set 128 columns for S, then dP.  dkv: P
// and dS overwrite S and dP as they are made, dP follows the product that reads P, and the next S the one that reads dS.  dq: 64
// more columns for dS, so that dP is formed while the exponentials run, and the next S as soon as dP has been read.
// P and dS are rounded to bf16 (relative 2^-8 at most); everything else is fp32.
//
// Measured (8192 rows, one sequence): 16 heads of 64 534 us, 16 query and 4 key heads of 128 745 us, 644 and 923 TFLOP/s counted
// as five products over the visible pairs; eleven documents in 8192 rows, 16 heads of 64: 145 us.  Bound at D = 128 by the tensor
// pipe (65 % busy over both kinds) and its latencies, at D = 64 by the exponentials and the instructions around them: products
// with 64 columns take as long as ones with 128.
//
// A first small kernel forms delta from o and the rest that its rounding left: where a row sees few keys ds is a small difference
// of dp and delta (zero for a row that sees itself alone), and the rounding of o alone would be most of the gradients' error (up
// to 3.9e-3 of dq's norm over documents of some ten tokens, 2.6e-3 with the rest).  It leaves -delta and -lse in base 2 (-inf for
// rows without keys and for the padding of the last tile, which makes their weights zero; NaN where fp32 does not hold lse to
// within an octave, as weights would be off by that: the gradients of such a row and of the keys that it sees are NaN).
#include "packed.cuh"

using namespace packed;

namespace {

constexpr int MORE = 4;

// aux: [2][Hq][Tp] fp32 (-lse in base 2, -delta), Tp = T rounded up to whole tiles
template <int LANES>
__global__ void __launch_bounds__(256) packed_delta_kernel(const bf16* __restrict__ o, const bf16* __restrict__ o_lo,
                                                           const bf16* __restrict__ go, long long g_rs,
                                                           long long g_hs, const float* __restrict__ lse, float* __restrict__ aux,
                                                           const int* __restrict__ cu, int nseq, int T, int Tp, int Hq, int D) {
  // one head, ROWS rows: LANES threads (8 dims each) take a row, MORE rows whose loads are in flight together, and the rows of
  // a warp's groups follow one another, so the row vectors are read and written in whole sectors: 12.3 us at 8192 rows of 16
  // heads of 64 with a cold cache (50 MB), 19.7 with the heads of a row in a warp
  constexpr int GROUPS = 256 / LANES, ROWS = GROUPS * MORE;
  const int h = blockIdx.x % Hq, row0 = blockIdx.x / Hq * ROWS + threadIdx.x / LANES;
  const int sub = threadIdx.x % LANES, begin = __ldg(cu), end = __ldg(cu + nseq);
  uint4 a[MORE], l[MORE], b[MORE];
  float L[MORE];
  bool inside[MORE];
#pragma unroll
  for (int k = 0; k < MORE; ++k) {
    const long long row = row0 + k * GROUPS;              // below Tp, a multiple of ROWS
    inside[k] = row < T && row >= begin && row < end;     // padding rows may hold anything
    a[k] = l[k] = b[k] = make_uint4(0, 0, 0, 0);
    if (inside[k] && sub * 8 < D) {
      a[k] = *reinterpret_cast<const uint4*>(o + (row * Hq + h) * D + sub * 8);
      if (o_lo) l[k] = *reinterpret_cast<const uint4*>(o_lo + (row * Hq + h) * D + sub * 8);
      b[k] = *reinterpret_cast<const uint4*>(go + row * g_rs + h * g_hs + sub * 8);
    }
    L[k] = inside[k] && sub == 0 ? lse[(long long)h * T + row] : -INFINITY;
  }
#pragma unroll
  for (int k = 0; k < MORE; ++k) {
    const uint32_t x[4] = {a[k].x, a[k].y, a[k].z, a[k].w}, z[4] = {l[k].x, l[k].y, l[k].z, l[k].w},
                   y[4] = {b[k].x, b[k].y, b[k].z, b[k].w};
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 p = unpack_bf16(x[i]), r = unpack_bf16(z[i]), q = unpack_bf16(y[i]);
      s = fmaf(p.x + r.x, q.x, s);
      s = fmaf(p.y + r.y, q.y, s);
    }
#pragma unroll
    for (int i = LANES / 2; i > 0; i >>= 1) s += __shfl_xor_sync(0xffffffffu, s, i);
    if (sub == 0) {
      const long long at = (long long)h * Tp + row0 + k * GROUPS;
      const float n = -L[k] * LOG2E;
      aux[at] = n == INFINITY ? -INFINITY : fabsf(n) <= FAR ? n : NAN;
      aux[(long long)Hq * Tp + at] = -s;
    }
  }
}

struct Geo {
  const int* cu;
  const float* aux;
  int nseq, T, Tp, Hq, Hkv, group, D, window, tiles;
  float scale, scale_log2;
};

__device__ __forceinline__ void load_bulk(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
               "r"(bytes), "r"(bar)
               : "memory");
}

// one row of a gradient: DH columns of tensor memory, scaled, to D bf16
template <int DH>
__device__ __forceinline__ void store_row(uint32_t taddr, bf16* dst, int D, float scale, bool live) {
#pragma unroll
  for (int c = 0; c < DH / 32; ++c) {
    uint32_t r[32];
    tmem_ld32(taddr + 32 * c, r);
    tmem_ld_wait();
    if (!live) continue;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      uint32_t w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        w[i] = pack_bf16(__uint_as_float(r[16 * u + 2 * i]) * scale, __uint_as_float(r[16 * u + 2 * i + 1]) * scale);
      const int d0 = 32 * c + 16 * u;
      if (d0 + 16 <= D && (D & 15) == 0) {
        st_global_32(dst + d0, w);
      } else if (d0 < D) {
        *reinterpret_cast<uint4*>(dst + d0) = make_uint4(w[0], w[1], w[2], w[3]);
        if (d0 + 8 < D) *reinterpret_cast<uint4*>(dst + d0 + 8) = make_uint4(w[4], w[5], w[6], w[7]);
      }
    }
  }
}

template <int DH>
struct Cfg {
  static constexpr int SETS = DH == 128 ? 2 : 1;           // steps in work in a CTA
  static constexpr int NT = (SETS + 1) * 128, ISSUE = SETS * 4, LOAD = ISSUE + 1, COLS = SETS * 256;
  static constexpr int TB = TILE * DH * 2;
  // rings of single tiles: A (dkv: queries, dq: keys) is read by the first and by the last product of a step, B by those between
  static constexpr int NA = SETS + 1, NB = 2;
  static constexpr int own_off = 0, a_off = 2 * TB, b_off = a_off + NA * TB;
  // dkv: 128 -delta per tile of A and 128 -lse per tile of B, so each lies there until the math warps have read it
  static constexpr int aux_off = b_off + NB * TB;
  static constexpr int bar_off = aux_off + (NA + NB) * 512;
  static constexpr int total = bar_off + 304;
  static __device__ __forceinline__ int set(int i) { return i % SETS; }                       // of step i
  static __device__ __forceinline__ uint32_t phase(int i) { return (uint32_t)(i / SETS) & 1; }  // of its set's barriers
};
static_assert(Cfg<128>::total <= 227 * 1024 && Cfg<64>::total <= 113 * 1024, "shared memory");

// P = exp2(s * scale + nl) in place, nl = -lse.  All on the special-function unit: a share of them on the FMA pipe as in the
// forward pass was slower here (8192 x 16 heads of 64: none 517, one of eight pairs 525, two 534 us; half a row per thread and
// twice the warps 551 us).
__device__ __forceinline__ void exponential_pair(uint32_t& a, uint32_t& b, f32x2 sc, f32x2 nl) {
  float y0, y1;
  split(fma2(pair(__uint_as_float(a), __uint_as_float(b)), sc, nl), y0, y1);
  a = __float_as_uint(ex2(y0));
  b = __float_as_uint(ex2(y1));
}
// a row per thread, 32 of its columns
__device__ __forceinline__ void exponentials(uint32_t (&x)[32], float scale, f32x2 nl) {
  const f32x2 sc = pair(scale, scale);
#pragma unroll
  for (int i = 0; i < 16; ++i) exponential_pair(x[2 * i], x[2 * i + 1], sc, nl);
}
// fragments of 32 rows and 128 columns; nl: this thread's pair of every 8 columns
__device__ __forceinline__ void exponentials(uint32_t (&x)[2][64], float scale, const f32x2* nl) {
  const f32x2 sc = pair(scale, scale);
#pragma unroll
  for (int u = 0; u < 16; ++u) {
    const f32x2 n = nl[4 * u];
#pragma unroll
    for (int v = 0; v < 4; ++v) exponential_pair(x[v >> 1][4 * u + 2 * (v & 1)], x[v >> 1][4 * u + 2 * (v & 1) + 1], sc, n);
  }
}
// columns outside [lo, hi] to zero; c0: the first of the 32 columns
__device__ __forceinline__ void clear_hidden(uint32_t (&x)[32], int c0, int lo, int hi) {
  const uint32_t seen = range_bits(c0, lo, hi);
#pragma unroll
  for (int i = 0; i < 32; ++i) x[i] = seen & (1u << i) ? x[i] : 0u;
}
__device__ __forceinline__ void store_packed(uint32_t taddr, const uint32_t (&x)[32]) {
  uint32_t w[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) w[i] = pack_bf16(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1]));
  tmem_st16(taddr, w);
}
// dS = P (dP - delta) in place, nd = -delta
__device__ __forceinline__ void scale_pair(uint32_t& a, uint32_t& b, uint32_t d0, uint32_t d1, f32x2 nd) {
  float s0, s1;
  split(mul2(pair(__uint_as_float(a), __uint_as_float(b)), add2(pair(__uint_as_float(d0), __uint_as_float(d1)), nd)), s0, s1);
  a = __float_as_uint(s0);
  b = __float_as_uint(s1);
}
// a math warp has read what it wanted of tensor memory
__device__ __forceinline__ void release(uint32_t bar, int lane) {
  tc_fence_before();
  __syncwarp();
  if (lane == 0) mbar_arrive(bar);
}
// what a math warp has written to tensor memory is there for the products
__device__ __forceinline__ void hand_over(uint32_t bar, int lane) {
  tmem_st_wait();
  tc_fence_before();
  __syncwarp();
  if (lane == 0) mbar_arrive(bar);
}

// ---------------------------------------------------------------------------------------------------------------------------
template <int DH>
__device__ __forceinline__ void keys_and_values(const CUtensorMap& tmQ, const CUtensorMap& tmK, const CUtensorMap& tmV,
                                                const CUtensorMap& tmG, bf16* __restrict__ dk, bf16* __restrict__ dv, const Geo& g,
                                                int block, int* __restrict__ gerr) {
  using C = Cfg<DH>;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t base = smem_u32(smem);
  if (base & 1023u) {
    if (threadIdx.x == 0) atomicExch(gerr, 2);
    return;
  }
  const uint32_t bar0 = base + C::bar_off;
  // barriers: own, done, drained, sfull[2], pfull[2], dpfull[2], dsfull[2], then the rings'
  const uint32_t own = bar0, done = bar0 + 8, drained = bar0 + 16;
  auto sfull = [&](int a) { return bar0 + 24 + 8u * a; };
  auto pfull = [&](int a) { return bar0 + 40 + 8u * a; };
  auto dpfull = [&](int a) { return bar0 + 56 + 8u * a; };
  auto dsfull = [&](int a) { return bar0 + 72 + 8u * a; };
  auto qfull = [&](int i) { return bar0 + 88 + 8u * (i % C::NA); };
  auto qempty = [&](int i) { return bar0 + 88 + 8u * (C::NA + i % C::NA); };
  auto gfull = [&](int i) { return bar0 + 88 + 8u * (2 * C::NA + i % C::NB); };
  auto gempty = [&](int i) { return bar0 + 88 + 8u * (2 * C::NA + C::NB + i % C::NB); };
  auto qphase = [](int i) { return (uint32_t)(i / C::NA) & 1; };
  auto gphase = [](int i) { return (uint32_t)(i / C::NB) & 1; };
  volatile uint32_t* tslot = reinterpret_cast<volatile uint32_t*>(smem + C::bar_off + 280);
  volatile int* serr = reinterpret_cast<volatile int*>(smem + C::bar_off + 288);
  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  // the first keys of a long sequence are seen by the most queries: they come first
  const int kh = block % g.Hkv, kt = block / g.Hkv, key0 = kt * TILE;
  const uint32_t sK = base + C::own_off, sV = sK + C::TB;
  auto sQ = [&](int i) { return base + C::a_off + (i % C::NA) * C::TB; };
  auto sG = [&](int i) { return base + C::b_off + (i % C::NB) * C::TB; };
  auto load_queries = [&](int i, int h, int q0) {
    mbar_expect_tx(qfull(i), C::TB + 512);
    load_tile<DH>(sQ(i), &tmQ, qfull(i), h, q0);
    load_bulk(base + C::aux_off + (i % C::NA) * 512, g.aux + (long long)(g.Hq + h) * g.Tp + q0, 512, qfull(i));
  };
  auto load_gradients = [&](int i, int h, int q0) {
    mbar_expect_tx(gfull(i), C::TB + 512);
    load_tile<DH>(sG(i), &tmG, gfull(i), h, q0);
    load_bulk(base + C::aux_off + (C::NA + i % C::NB) * 512, g.aux + (long long)h * g.Tp + q0, 512, gfull(i));
  };
  if (warp == C::LOAD) {
    if (elect_one()) {
      *serr = 0;
      mbar_init(own, 1);
      mbar_init(done, 1);
      mbar_init(drained, 1);
      for (int a = 0; a < 2; ++a) {
        mbar_init(sfull(a), 1);
        mbar_init(pfull(a), 4);
        mbar_init(dpfull(a), 1);
        mbar_init(dsfull(a), 4);
      }
      for (int i = 0; i < C::NA; ++i) { mbar_init(qfull(i), 1); mbar_init(qempty(i), 1); }
      for (int i = 0; i < C::NB; ++i) { mbar_init(gfull(i), 1); mbar_init(gempty(i), 1); }
      fence_barrier_init();
      // what does not depend on the sequences: the keys and the queries of their own tile
      mbar_expect_tx(own, 2 * C::TB);
      load_tile<DH>(sK, &tmK, own, kh, key0);
      load_queries(0, kh * g.group, key0);
      load_tile<DH>(sV, &tmV, own, kh, key0);
      load_gradients(0, kh * g.group, key0);
    }
    __syncwarp();
  }
  if (warp == C::ISSUE) tmem_alloc(tslot, C::COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tm = uniform(*tslot);
  auto tX = [&](int a) { return tm + a * TILE; };                                   // S, P, dP, dS
  const uint32_t tdV = tm + C::SETS * TILE, tdK = tdV + DH;
  const int last = last_query(g.cu, g.nseq, g.window, g.T, min(g.T, key0 + TILE) - 1);
  const int nq = uniform(max(kt, last / TILE)) - kt + 1, steps = nq * g.group;     // query tiles kt .. kt + nq - 1 of each head

  if (warp >= C::ISSUE) {
    // 384 threads launch with 168 registers each, 2 x 216 + 72 = 3 x 168; 256 (twice on an SM) with 128, 216 + 40 = 2 x 128
    if (C::SETS == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;"); else asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (warp == C::LOAD) {
      int i = 1, qi = nq == 1 ? 0 : 1, h = kh * g.group + (nq == 1);        // step 0 is on its way
      for (; i < steps && !*serr; ++i) {
        const int q0 = (kt + qi) * TILE;
        wait(qempty(i), qphase(i) ^ 1, serr);
        if (elect_one()) load_queries(i, h, q0);
        wait(gempty(i), gphase(i) ^ 1, serr);
        if (elect_one()) load_gradients(i, h, q0);
        if (++qi == nq) { qi = 0; ++h; }
      }
      if (*serr) {          // a wait ran out: let the copies in flight land before the CTA ends
        volatile int ignore = 0;
        mbar_wait(own, 0, &ignore);
        for (int u = max(0, i - C::NA); u < i; ++u) mbar_wait(qfull(u), qphase(u), &ignore);
        for (int u = max(0, i - C::NB); u < i; ++u) mbar_wait(gfull(u), gphase(u), &ignore);
      }
    } else if (warp == C::ISSUE) {
      constexpr uint32_t idS = mma_desc<bf16>(TILE, TILE, 0, 0), idG = mma_desc<bf16>(TILE, DH, 0, 1);
      const int begin = max(0, __ldg(g.cu)), end = min(g.T, __ldg(g.cu + g.nseq));
      auto clean = [&](int off, int q0) {                // the padding rows of a tile that has just arrived
        if (q0 < begin || q0 + TILE > end) blank_rows<DH>(smem + off, q0, begin, end, lane);
      };
      auto scores = [&](int i, int q0) {                 // S^T = K Q_i^T
        wait(qfull(i), qphase(i), serr);
        clean(C::a_off + (i % C::NA) * C::TB, q0);
        tc_fence_after();
        if (elect_one()) {
          const uint64_t k = desc_dims(sK, 0), q = desc_dims(sQ(i), 0);
#pragma unroll
          for (int u = 0; u < DH / 16; ++u) umma_bf16(tX(C::set(i)), k + dims_step(u), q + dims_step(u), idS, u != 0);
          umma_commit(sfull(C::set(i)));
        }
        __syncwarp();
      };
      auto dscores = [&](int i) {                        // dP^T = V dO_i^T
        tc_fence_after();
        if (elect_one()) {
          const uint64_t v = desc_dims(sV, 0), go = desc_dims(sG(i), 0);
#pragma unroll
          for (int u = 0; u < DH / 16; ++u) umma_bf16(tX(C::set(i)), v + dims_step(u), go + dims_step(u), idS, u != 0);
          umma_commit(dpfull(C::set(i)));
          umma_commit(gempty(i));
        }
        __syncwarp();
      };
      auto values = [&](int i) {                         // dV += P^T dO_i
        tc_fence_after();
        if (elect_one()) {
          const uint64_t go = desc_rows(sG(i), 0);
#pragma unroll
          for (int u = 0; u < TILE / 16; ++u) umma_ts(tdV, tX(C::set(i)) + 8 * u, go + rows_step(u), idG, i > 0 || u != 0);
        }
        __syncwarp();
      };
      auto keys = [&](int i) {                           // dK += dS^T Q_i
        wait(dsfull(C::set(i)), C::phase(i), serr);
        tc_fence_after();
        if (elect_one()) {
          const uint64_t q = desc_rows(sQ(i), 0);
#pragma unroll
          for (int u = 0; u < TILE / 16; ++u) umma_ts(tdK, tX(C::set(i)) + 8 * u, q + rows_step(u), idG, i > 0 || u != 0);
          umma_commit(qempty(i));
          if (i + 1 == steps) umma_commit(done);
        }
        __syncwarp();
      };
      wait(own, 0, serr);
      int q0 = key0, ahead0 = key0;                      // first rows of the query tiles of step i and of the next scores
      auto next = [&](int v) { return v + TILE == key0 + nq * TILE ? key0 : v + TILE; };
      scores(0, ahead0);
      ahead0 = next(ahead0);
      if (C::SETS > 1 && steps > 1) { scores(1, ahead0); ahead0 = next(ahead0); }
      auto begin_step = [&](int i) {                     // P -> dV, and dP in its place behind it
        wait(gfull(i), gphase(i), serr);
        clean(C::b_off + (i % C::NB) * C::TB, q0);
        q0 = next(q0);
        wait(pfull(C::set(i)), C::phase(i), serr);
        values(i);
        dscores(i);
      };
      auto finish = [&](int i) {                         // dS -> dK, and the set's next scores
        keys(i);
        if (i + C::SETS < steps) { scores(i + C::SETS, ahead0); ahead0 = next(ahead0); }
      };
      if (C::SETS == 1) {
        for (int i = 0; i < steps; ++i) {
          begin_step(i);
          finish(i);
        }
      } else {
        // between the two halves of a step its set needs the tensor pipe's latency and the time to form dS: in this order the
        // other set's products fill it
        for (int i = 0; i < steps; i += 2) {
          begin_step(i);
          if (i > 0) finish(i - 1);
          finish(i);
          if (i + 1 < steps) begin_step(i + 1);
        }
        if (!(steps & 1)) finish(steps - 1);
      }
      drain_products(drained, serr);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    // Scores are read as MMA fragments (16 lanes x 256 bits): a thread holds four of its warp's 32 keys and every fourth pair of
    // queries, so it wants lse and delta of 32 queries instead of 128.  With a key per thread, handing every value of both to
    // every thread took as much of shared memory's bandwidth as two of the products (D = 128: 3000 cycles a step).
    const int a = warp >> 2, t4 = lane & 3, first = key0 + (warp & 3) * 32, own_key = first + lane;
    const uint32_t tl = (uint32_t)((warp & 3) * 32) << 16, lower = 16u << 16;
    const uint32_t x_addr = tX(a) + tl;
    const int own_hi = own_key < g.T ? last_query(g.cu, g.nseq, g.window, g.T, own_key) : own_key - 1;
    const int w_hi = __shfl_sync(0xffffffffu, own_hi, 0), w_key = first + 31;         // hi ascends with the key
    int hi[2][2];                                                                     // of key first + 16 h + 8 e + lane / 4
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int e = 0; e < 2; ++e) hi[h][e] = __shfl_sync(0xffffffffu, own_hi, 16 * h + 8 * e + (lane >> 2));
    int qi = a % nq;
    for (int i = a; i < steps; i += C::SETS) {
      const uint32_t ph = C::phase(i);
      const int q0 = (kt + qi) * TILE;
      qi = (qi + C::SETS) % nq;
      const f32x2* ndelta = reinterpret_cast<const f32x2*>(smem + C::aux_off + (i % C::NA) * 512) + t4;
      const f32x2* nlse = reinterpret_cast<const f32x2*>(smem + C::aux_off + (C::NA + i % C::NB) * 512) + t4;
      wait(sfull(a), ph, serr);
      wait(qfull(i), qphase(i), serr);                     // delta arrived with the queries
      wait(gfull(i), gphase(i), serr);                     // and lse with the output's gradient
      tc_fence_after();
      uint32_t x[2][64];
      tmem_ld_16x256b_x16(x_addr, x[0]);
      tmem_ld_16x256b_x16(x_addr + lower, x[1]);
      tmem_ld_wait();
      const bool mask = q0 < w_key || q0 + TILE - 1 > w_hi;
      auto clear = [&]() {                                 // queries that do not see the key
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int lo_c = first + 16 * h + 8 * e + (lane >> 2) - q0 - 2 * t4, hi_c = hi[h][e] - q0 - 2 * t4;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const uint32_t seen = range_bits(32 * c, lo_c, hi_c);
#pragma unroll
              for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                  uint32_t& v = x[h][16 * c + 4 * u + 2 * e + w];
                  v = seen & (1u << (8 * u + w)) ? v : 0u;
                }
            }
          }
      };
      auto store = [&]() {                                 // as the 16-bit operand of the next product
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t w[32];
#pragma unroll
          for (int u = 0; u < 32; ++u) w[u] = pack_bf16(__uint_as_float(x[h][2 * u]), __uint_as_float(x[h][2 * u + 1]));
          tmem_st_16x128b_x16(x_addr + h * lower, w);
        }
      };
      if (mask) {                                          // two branches with the same exponentials: see queries_only
        exponentials(x, g.scale_log2, nlse);
        clear();
      } else {
        exponentials(x, g.scale_log2, nlse);
      }
      store();
      hand_over(pfull(a), lane);
      wait(dpfull(a), ph, serr);
      tc_fence_after();
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t d[64];
        tmem_ld_16x256b_x16(x_addr + h * lower, d);
        tmem_ld_wait();
#pragma unroll
        for (int u = 0; u < 16; ++u) {
          const f32x2 nd = ndelta[4 * u];
#pragma unroll
          for (int e = 0; e < 2; ++e) scale_pair(x[h][4 * u + 2 * e], x[h][4 * u + 2 * e + 1], d[4 * u + 2 * e], d[4 * u + 2 * e + 1], nd);
        }
      }
      if (mask) clear();                                   // 0 x (what a padding row's product left) is not zero
      store();
      hand_over(dsfull(a), lane);
    }
    wait(done, 0, serr);
    tc_fence_after();
    const long long off = ((long long)own_key * g.Hkv + kh) * g.D;
    if (a == 0) store_row<DH>(tdV + tl, dv + off, g.D, 1.f, own_key < g.T);
    if (a == C::SETS - 1) store_row<DH>(tdK + tl, dk + off, g.D, g.scale, own_key < g.T);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == C::ISSUE) tmem_dealloc(tm, C::COLS);
  if (threadIdx.x == 0 && *serr) atomicExch(gerr, 1);
}

// ---------------------------------------------------------------------------------------------------------------------------
template <int DH>
__device__ __forceinline__ void queries_only(const CUtensorMap& tmQ, const CUtensorMap& tmK, const CUtensorMap& tmV,
                                             const CUtensorMap& tmG, bf16* __restrict__ dq, const Geo& g, int block,
                                             int* __restrict__ gerr) {
  using C = Cfg<DH>;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t base = smem_u32(smem);
  if (base & 1023u) {
    if (threadIdx.x == 0) atomicExch(gerr, 2);
    return;
  }
  const uint32_t bar0 = base + C::bar_off;
  // barriers: own, done, drained, sfull[2], sread[2], dqdone[2], dpfull[2], dsfull[2], dpread[2], then the rings'
  const uint32_t own = bar0, done = bar0 + 8, drained = bar0 + 16;
  auto sfull = [&](int a) { return bar0 + 24 + 8u * a; };
  auto sread = [&](int a) { return bar0 + 40 + 8u * a; };
  auto dqdone = [&](int a) { return bar0 + 56 + 8u * a; };
  auto dpfull = [&](int a) { return bar0 + 72 + 8u * a; };
  auto dsfull = [&](int a) { return bar0 + 88 + 8u * a; };
  auto dpread = [&](int a) { return bar0 + 104 + 8u * a; };
  auto kfull = [&](int i) { return bar0 + 120 + 8u * (i % C::NA); };
  auto kempty = [&](int i) { return bar0 + 120 + 8u * (C::NA + i % C::NA); };
  auto vfull = [&](int i) { return bar0 + 120 + 8u * (2 * C::NA + i % C::NB); };
  auto vempty = [&](int i) { return bar0 + 120 + 8u * (2 * C::NA + C::NB + i % C::NB); };
  auto kphase = [](int i) { return (uint32_t)(i / C::NA) & 1; };
  auto vphase = [](int i) { return (uint32_t)(i / C::NB) & 1; };
  volatile uint32_t* tslot = reinterpret_cast<volatile uint32_t*>(smem + C::bar_off + 280);
  volatile int* serr = reinterpret_cast<volatile int*>(smem + C::bar_off + 288);
  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int h = block % g.Hq, qt = g.tiles - 1 - block / g.Hq, row0 = qt * TILE;
  const uint32_t sQ = base + C::own_off, sG = sQ + C::TB;
  auto sK = [&](int i) { return base + C::a_off + (i % C::NA) * C::TB; };
  auto sV = [&](int i) { return base + C::b_off + (i % C::NB) * C::TB; };
  const int kh = h / g.group;                              // key blocks from the diagonal down
  auto load_keys = [&](int i) {
    mbar_expect_tx(kfull(i), C::TB);
    load_tile<DH>(sK(i), &tmK, kfull(i), kh, (qt - i) * TILE);
  };
  auto load_values = [&](int i) {
    mbar_expect_tx(vfull(i), C::TB);
    load_tile<DH>(sV(i), &tmV, vfull(i), kh, (qt - i) * TILE);
  };
  if (warp == C::LOAD) {
    if (elect_one()) {
      *serr = 0;
      mbar_init(own, 1);
      mbar_init(done, 1);
      mbar_init(drained, 1);
      for (int a = 0; a < 2; ++a) {
        mbar_init(sfull(a), 1);
        mbar_init(sread(a), 4);
        mbar_init(dqdone(a), 1);
        mbar_init(dpfull(a), 1);
        mbar_init(dsfull(a), 4);
        mbar_init(dpread(a), 4);
      }
      for (int i = 0; i < C::NA; ++i) { mbar_init(kfull(i), 1); mbar_init(kempty(i), 1); }
      for (int i = 0; i < C::NB; ++i) { mbar_init(vfull(i), 1); mbar_init(vempty(i), 1); }
      fence_barrier_init();
      mbar_expect_tx(own, 2 * C::TB);
      load_tile<DH>(sQ, &tmQ, own, h, row0);
      load_keys(0);
      load_tile<DH>(sG, &tmG, own, h, row0);
      load_values(0);
    }
    __syncwarp();
  }
  if (warp == C::ISSUE) tmem_alloc(tslot, C::COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tm = uniform(*tslot);
  auto tX = [&](int a) { return tm + a * TILE; };                                   // S, then dP
  auto tDS = [&](int a) { return tm + C::SETS * TILE + DH + a * 64; };
  const uint32_t tdQ = tm + C::SETS * TILE;
  const int steps = qt - uniform(min(qt, first_key(g.cu, g.nseq, g.window, row0) / TILE)) + 1;

  if (warp >= C::ISSUE) {
    if (C::SETS == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;"); else asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (warp == C::LOAD) {
      int i = 1;                                           // step 0 is on its way
      for (; i < steps && !*serr; ++i) {
        wait(kempty(i), kphase(i) ^ 1, serr);
        if (elect_one()) load_keys(i);
        wait(vempty(i), vphase(i) ^ 1, serr);
        if (elect_one()) load_values(i);
      }
      if (*serr) {
        volatile int ignore = 0;
        mbar_wait(own, 0, &ignore);
        for (int u = max(0, i - C::NA); u < i; ++u) mbar_wait(kfull(u), kphase(u), &ignore);
        for (int u = max(0, i - C::NB); u < i; ++u) mbar_wait(vfull(u), vphase(u), &ignore);
      }
    } else if (warp == C::ISSUE) {
      constexpr uint32_t idS = mma_desc<bf16>(TILE, TILE, 0, 0), idG = mma_desc<bf16>(TILE, DH, 0, 1);
      const int begin = max(0, __ldg(g.cu)), end = min(g.T, __ldg(g.cu + g.nseq));
      auto scores = [&](int i) {                         // S = Q K_i^T
        const int k0 = (qt - i) * TILE;
        wait(kfull(i), kphase(i), serr);
        if (k0 < begin || k0 + TILE > end) blank_rows<DH>(smem + C::a_off + (i % C::NA) * C::TB, k0, begin, end, lane);
        tc_fence_after();
        if (elect_one()) {
          const uint64_t q = desc_dims(sQ, 0), k = desc_dims(sK(i), 0);
#pragma unroll
          for (int u = 0; u < DH / 16; ++u) umma_bf16(tX(C::set(i)), q + dims_step(u), k + dims_step(u), idS, u != 0);
          umma_commit(sfull(C::set(i)));
        }
        __syncwarp();
      };
      auto dscores = [&](int i) {                        // dP = dO V_i^T, once S has been read
        wait(vfull(i), vphase(i), serr);
        wait(sread(C::set(i)), C::phase(i), serr);
        tc_fence_after();
        if (elect_one()) {
          const uint64_t go = desc_dims(sG, 0), v = desc_dims(sV(i), 0);
#pragma unroll
          for (int u = 0; u < DH / 16; ++u) umma_bf16(tX(C::set(i)), go + dims_step(u), v + dims_step(u), idS, u != 0);
          umma_commit(dpfull(C::set(i)));
          umma_commit(vempty(i));
        }
        __syncwarp();
      };
      auto queries = [&](int i) {                        // dQ += dS K_i
        wait(dsfull(C::set(i)), C::phase(i), serr);
        tc_fence_after();
        if (elect_one()) {
          const uint64_t k = desc_rows(sK(i), 0);
#pragma unroll
          for (int u = 0; u < TILE / 16; ++u) umma_ts(tdQ, tDS(C::set(i)) + 8 * u, k + rows_step(u), idG, i > 0 || u != 0);
          umma_commit(kempty(i));
          umma_commit(dqdone(C::set(i)));
          if (i + 1 == steps) umma_commit(done);
        }
        __syncwarp();
      };
      wait(own, 0, serr);
      scores(0);
      if (C::SETS > 1 && steps > 1) scores(1);
      constexpr int LAG = C::SETS - 1;                   // with two sets, the other one's last step is in between
      for (int i = 0; i < steps; ++i) {
        dscores(i);
        const int e = i - LAG;                           // dP read -> the set's next S, and its dS -> dQ
        if (e >= 0) {
          if (e + C::SETS < steps) {
            wait(dpread(C::set(e)), C::phase(e), serr);
            scores(e + C::SETS);
          }
          queries(e);
        }
      }
      if (LAG) queries(steps - 1);
      drain_products(drained, serr);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int a = warp >> 2, row = row0 + (warp & 3) * 32 + lane;
    const uint32_t tl = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t x_addr = tX(a) + tl, ds_addr = tDS(a) + tl;
    const int lo = row < g.T ? first_key(g.cu, g.nseq, g.window, row) : row + 1;
    const int w_lo = __shfl_sync(0xffffffffu, lo, 31), w_row = row - lane;
    const float L = g.aux[(long long)h * g.Tp + row], D = g.aux[((long long)g.Hq + h) * g.Tp + row];
    const f32x2 nl = pair(L, L), nd = pair(D, D);
    for (int i = a; i < steps; i += C::SETS) {
      const uint32_t ph = C::phase(i);
      const int k0 = (qt - i) * TILE;
      wait(sfull(a), ph, serr);
      tc_fence_after();
      uint32_t x[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld32(x_addr + 32 * c, x[c]);
      tmem_ld_wait();
      release(sread(a), lane);
      const bool mask = k0 < w_lo || k0 + TILE - 1 > w_row;
      const int c_lo = lo - k0, c_hi = row - k0;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        // The exponentials belong before the wait for dP, which they hide.  Only results that come out of a branch stay there:
        // without one the compiler moves them to their use behind the wait (8192 x 16 heads of 64: dq 293 against 237 us).
        if (mask) exponentials(x[c], g.scale_log2, nl);
        else exponentials(x[c], g.scale_log2, nl);
      }
      wait(dpfull(a), ph, serr);
      tc_fence_after();
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t d[2][32];
        tmem_ld32(x_addr + 64 * half, d[0]);
        tmem_ld32(x_addr + 64 * half + 32, d[1]);
        tmem_ld_wait();
        if (half) release(dpread(a), lane);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int c = 2 * half + u;
#pragma unroll
          for (int w = 0; w < 32; w += 2) scale_pair(x[c][w], x[c][w + 1], d[u][w], d[u][w + 1], nd);
          if (mask) clear_hidden(x[c], 32 * c, c_lo, c_hi);  // 0 x (what a padding row's product left) is not zero
        }
      }
      if (i >= C::SETS) {                                  // the last dS of this set has been read
        wait(dqdone(a), C::phase(i) ^ 1, serr);
        tc_fence_after();
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) store_packed(ds_addr + 16 * c, x[c]);
      hand_over(dsfull(a), lane);
    }
    wait(done, 0, serr);
    tc_fence_after();
    if (a == 0) store_row<DH>(tdQ + tl, dq + ((long long)row * g.Hq + h) * g.D, g.D, g.scale, row < g.T);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == C::ISSUE) tmem_dealloc(tm, C::COLS);
  if (threadIdx.x == 0 && *serr) atomicExch(gerr, 1);
}

// One launch for both: the dkv blocks, which have more to do, come first, and dq blocks fill the SMs that they leave.
template <int DH>
__global__ void __launch_bounds__(Cfg<DH>::NT, 3 - Cfg<DH>::SETS) packed_bwd_kernel(
    const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
    const __grid_constant__ CUtensorMap tmG, bf16* __restrict__ dq, bf16* __restrict__ dk, bf16* __restrict__ dv,
    const __grid_constant__ Geo g, int* __restrict__ gerr) {
  const int n = g.tiles * g.Hkv, block = blockIdx.x;
  if (block < n) keys_and_values<DH>(tmQ, tmK, tmV, tmG, dk, dv, g, block, gerr);
  else queries_only<DH>(tmQ, tmK, tmV, tmG, dq, g, block - n, gerr);
}

template <int DH>
int launch(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const CUtensorMap& mg, bf16* dq, bf16* dk, bf16* dv,
           const Geo& g, int* err, cudaStream_t st) {
  static std::atomic<unsigned long long> set{0};
  if (int rc = allow_smem(packed_bwd_kernel<DH>, Cfg<DH>::total, set)) return rc;
  packed_bwd_kernel<DH><<<(unsigned)(g.tiles * (g.Hkv + g.Hq)), Cfg<DH>::NT, Cfg<DH>::total, st>>>(mq, mk, mv, mg, dq, dk, dv, g, err);
  DMB_CHECK_LAUNCH();
  return 0;
}

}  // namespace

// bf16: go (gradient of o) [T, Hq, D] and q, k, v by strides as in dmb_packed_attn_fwd; o, dq [T, Hq, D], dk, dv [T, Hkv, D]
// contiguous, o_lo like o or null; lse [Hq, T]; aux fp32 [2, Hq, Tp] with Tp = T rounded up to a multiple of 128.  All gradient rows are written.
extern "C" int dmb_packed_attn_bwd(const void* go, long long g_rs, long long g_hs, const void* q, long long q_rs, long long q_hs,
                                   const void* k, long long k_rs, long long k_hs, const void* v, long long v_rs, long long v_hs,
                                   const void* o, const void* o_lo, const float* lse, const int* cu, int nseq, float* aux, void* dq, void* dk,
                                   void* dv, int T, int Hq, int Hkv, int D, int window, float scale, int* err, void* stream) {
  if (T <= 0) return 0;
  if (D <= 0 || D > 128 || (D & 7) || Hkv <= 0 || Hq % Hkv || nseq < 0) return -1;
  CUtensorMap mq, mk, mv, mg;
  int rc = bind_context();
  if (rc == 0) rc = make_map_rows(&mq, q, D, Hq, T, q_rs, q_hs);
  if (rc == 0) rc = make_map_rows(&mk, k, D, Hkv, T, k_rs, k_hs);
  if (rc == 0) rc = make_map_rows(&mv, v, D, Hkv, T, v_rs, v_hs);
  if (rc == 0) rc = make_map_rows(&mg, go, D, Hq, T, g_rs, g_hs);
  if (rc) return rc;
  const int tiles = (int)(((long long)T + TILE - 1) / TILE);
  if ((long long)tiles * (Hq + Hkv) > 0x7fffffffLL) return -1;
  const Geo g{cu, aux, nseq, T, tiles * TILE, Hq, Hkv, Hq / Hkv, D, window, tiles, scale, scale * LOG2E};
  cudaStream_t st = (cudaStream_t)stream;
  const long long rows = (long long)g.Tp * Hq;
  const unsigned blocks = (unsigned)(rows / (256 / (D <= 64 ? 8 : 16) * MORE));     // whole ones: Tp is a multiple of 128
  auto delta = D <= 64 ? packed_delta_kernel<8> : packed_delta_kernel<16>;
  delta<<<blocks, 256, 0, st>>>((const bf16*)o, (const bf16*)o_lo, (const bf16*)go, g_rs, g_hs, lse, aux, cu, nseq, T, g.Tp, Hq, D);
  DMB_CHECK_LAUNCH();
  return D <= 64 ? launch<64>(mq, mk, mv, mg, (bf16*)dq, (bf16*)dk, (bf16*)dv, g, err, st)
                 : launch<128>(mq, mk, mv, mg, (bf16*)dq, (bf16*)dk, (bf16*)dv, g, err, st);
}
