// Causal attention over packed sequences, forward, on the 5th-generation tensor cores.
//
//   s_ij = scale q_i . k_j   for first_key(i) <= j <= i,   o_i = sum_j softmax(s_i)_j v_j,   lse_i = log sum_j exp s_ij
//
// q [T, Hq, D], k / v [T, Hkv, D], sequences packed one behind the other on the row axis (packed.cuh); query head h reads key
// head h / (Hq / Hkv).  A tile is 128 consecutive packed rows whatever sequences they belong to, so short sequences cost no
// padding: the keys a tile needs are one contiguous range, and each row masks to its own part of it.
//
// D = 128: one CTA per (head, pair of query tiles) on an SM; D = 64: one CTA per (head, query tile), two of them on an SM, which
// start and end independently of one another (tensor memory, 512 columns, holds two tiles either way).  Key blocks of 128
// stream through a shared-memory ring.  Per tile
//   four softmax warps (a thread owns a row = a lane of tensor memory), and per CTA
//   one warp that issues S = Q K^T, and O += P V with P in tensor memory, and one for the TMA loads.
// Scores stay in tensor memory only until the softmax has read them into registers, and P has columns of its own, so the next
// scores are formed while the exponentials of the last ones run.  D = 64: 128 columns S, 64 P, 64 O.  D = 128: the two tiles
// take turns with one S (128 + 2 x (64 P + 128 O)).  The turns cost little, since S is held for a product, its latency and one
// read, and they keep the two tiles half a block apart: one tile's exponentials run while the tensor pipe works for the other.
//
// Measured: 8192 rows of one sequence, 16 heads of 64: 190 us (722 TFLOP/s over the visible pairs); 16384 rows, 16 heads of 128:
// 895 us (1228 TFLOP/s, 75 % of the library product's measured rate); eleven documents in 8192 rows, where half of the
// blocks hold a border: 53 us.  128 x 128 exponentials take 1024 cycles of the special-function unit, as long as the products at
// D = 128 and twice as long at D = 64 (where no unit is full: special-function unit 54 %, issue slots 51 %, tensor pipe 35 %; a
// tile's next scores wait until the softmax has read the last).  So of every eight pairs EMU are computed by a polynomial on the FMA pipe
// (packed.cuh), in blocks without masked entries.  The running maximum is allowed to lag by up to 8 octaves (P <= 256, exact in
// the fp32 accumulator's range and no loss of relative precision in 16 bits): O is rescaled in tensor memory only when a row's
// maximum outgrows that, which after the first blocks is rare.  Sums are fp32; P is rounded to the operand type.
//
// Every mbarrier wait is bounded in time; on expiry the kernel raises a flag in global memory, stops waiting, lets its own
// copies land (bounded) and releases its tensor memory.
#include "packed.cuh"

using namespace packed;

namespace {

constexpr float LAG = 8.f;              // octaves
// Exponents are one FMA, the score in octaves minus the rounded maximum.  Up to 2^24 octaves that rounding is at most one octave
// and common to the row; beyond (FAR), the weights may leave the range of fp16 or fp32, and the row is computed again.

template <int DH>
struct Cfg {
  static constexpr int TILES = DH == 128 ? 2 : 1;
  static constexpr bool TURNS = TILES == 2;                // one S for both tiles
  static constexpr int NT = (TILES + 1) * 128, ISSUE = TILES * 4, LOAD = ISSUE + 1;      // threads; the issuing and loading warps
  static constexpr int COLS = TILES * 256;                 // tensor memory
  // pairs of eight on the FMA pipe; 8192 rows, 16 query heads and 16 key heads of 64 / 4 of 128: 0: 199.9 / 222.1,
  // 1: 194.1 / 229.1, 2: 191.1 / 232.8, 3: 190.9 / 236.3 us
  static constexpr int EMU = DH == 64 ? 2 : 0;
  static constexpr int P_OFF = TILE, O_OFF = TILE + TILES * 64;        // S, then P and O of each tile
  static constexpr int TB = TILE * DH * 2;                 // one tile
  static constexpr int SLOTS = 5;
  static constexpr int q_off = 0, ring_off = TILES * TB;
  static constexpr int bar_off = ring_off + SLOTS * TB;
  static constexpr int total = bar_off + 256;
};

struct Rows {                             // element (row, head, dim) at p[row * rs + head * hs + dim]
  const void* p;
  long long rs, hs;
};

struct Geo {
  const int* cu;
  int nseq, T, Hq, group, D, window, units;
  float scale_log2;
  Rows q, k, v;
};

// 32 weights of a row from 32 scores: exp2(s * scale - sub); returns their sum, leaves the packed columns in p
template <typename T, int EMU>
__device__ __forceinline__ f32x2 weights(const uint32_t (&x)[32], float scale, float sub, uint32_t (&p)[16]) {
  f32x2 sum[2] = {pair(0.f, 0.f), pair(0.f, 0.f)};
  const f32x2 sc = pair(scale, scale), sb = pair(-sub, -sub);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const f32x2 y = fma2(pair(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1])), sc, sb);
    float p0, p1;
    if ((i * EMU) % 8 + EMU > 7) {                          // EMU of eight, spread evenly
      ex2_pair(y, p0, p1);
    } else {
      split(y, p0, p1);
      p0 = ex2(p0);
      p1 = ex2(p1);
    }
    sum[i & 1] = add2(sum[i & 1], pair(p0, p1));
    p[i] = Elem<T>::pack(p0, p1);
  }
  return add2(sum[0], sum[1]);
}

// 16 dims of a row from d0 on, as far as the row has them (dims are a multiple of 8)
template <typename T>
__device__ __forceinline__ void store16(T* row, int d0, int D, const uint32_t (&w)[8]) {
  if (d0 + 16 <= D && (D & 15) == 0) {
    st_global_32(row + d0, w);
  } else if (d0 < D) {
    *reinterpret_cast<uint4*>(row + d0) = make_uint4(w[0], w[1], w[2], w[3]);
    if (d0 + 8 < D) *reinterpret_cast<uint4*>(row + d0 + 8) = make_uint4(w[4], w[5], w[6], w[7]);
  }
}

// One output row from the keys that it sees, at least one with a score above -inf; a whole warp: a lane scores one of 32 keys, then
// holds every 32nd dim.  Maximum and sum are its own: fp32 sums of another order than the tensor pipe's.
// The products run over blocks of 128 keys, where a weight of zero times an infinite or NaN value is NaN, so a row that does
// not see that value would get it all the same.  Rows whose scores are finite and whose outputs are not therefore end here,
// and rows of finite scores whose maximum is beyond FAR (every row of one sequence of 16384, 16 heads of 64: 275 ms),
// which costs the others up to 1 % (8192 mixed rows, 16 query and 4 key heads of 128: 78.4 against 79.6 us), and the smallest
// launches up to a microsecond of instruction fetches (731 rows, 16 heads of 64: 8.4 us with and without on some devices, 8.4
// against 9.5 on others).
template <typename T>
__device__ __forceinline__ void redo_row(const Geo& g, T* out, T* out_lo, float* lse, int h, int row, int lo) {
  const int lane = threadIdx.x & 31;
  const T* q = (const T*)g.q.p + row * g.q.rs + h * g.q.hs;
  const T* k = (const T*)g.k.p + h / g.group * g.k.hs;
  const T* v = (const T*)g.v.p + h / g.group * g.v.hs;
  float acc[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
#pragma unroll 1
  for (long long j0 = lo; j0 <= row; j0 += 32) {
    float s = -INFINITY;
    if (j0 + lane <= row) {
      s = 0.f;
#pragma unroll 2
      for (int d = 0; d < g.D; d += 8) {
        const uint4 a = *reinterpret_cast<const uint4*>(q + d), b = *reinterpret_cast<const uint4*>(k + (j0 + lane) * g.k.rs + d);
        const uint32_t x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 e = Elem<T>::unpack(x[i]), f = Elem<T>::unpack(y[i]);
          s = fmaf(e.x, f.x, s);
          s = fmaf(e.y, f.y, s);
        }
      }
    }
    float top = s;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (top > m) {
      const float f = ex2((m - top) * g.scale_log2);
      m = top;
      l *= f;
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] *= f;
    }
    const float w = m == -INFINITY ? 0.f : ex2((s - m) * g.scale_log2);
    l += w;
    const int n = (int)min(32LL, row + 1 - j0);
#pragma unroll 4
    for (int u = 0; u < n; ++u) {
      const float p = __shfl_sync(0xffffffffu, w, u);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (lane + 32 * i < g.D) acc[i] = fmaf(p, (float)v[(j0 + u) * g.v.rs + lane + 32 * i], acc[i]);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
  if (lse && lane == 0) lse[(long long)h * g.T + row] = fmaf(m, g.scale_log2, log2f(l)) * (1.f / LOG2E);
  l = 1.f / l;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (lane + 32 * i >= g.D) break;
    const long long at = ((long long)row * g.Hq + h) * g.D + lane + 32 * i;
    const float f = acc[i] * l;
    const T o = (T)f;
    out[at] = o;
    if (out_lo) out_lo[at] = (T)(f - (float)o);
  }
}

template <typename T, int DH>
__global__ void __launch_bounds__(Cfg<DH>::NT, 3 - Cfg<DH>::TILES) packed_fwd_kernel(
    const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
    T* __restrict__ out, T* __restrict__ out_lo, float* __restrict__ lse, const Geo g, int* __restrict__ gerr) {
  using C = Cfg<DH>;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t base = smem_u32(smem);
  if (base & 1023u) {
    if (threadIdx.x == 0) atomicExch(gerr, 2);
    return;
  }
  const uint32_t bar0 = base + C::bar_off;
  // barriers: qfull, sfull[2], sread[2], pfull[2], pvdone[2], drained, full[SLOTS], empty[SLOTS]
  const uint32_t qfull = bar0;
  auto sfull = [&](int a) { return bar0 + 8u * (1 + a); };
  auto sread = [&](int a) { return bar0 + 8u * (3 + a); };
  auto pfull = [&](int a) { return bar0 + 8u * (5 + a); };
  auto pvdone = [&](int a) { return bar0 + 8u * (7 + a); };
  const uint32_t drained = bar0 + 8u * 9;
  auto full = [&](int s) { return bar0 + 8u * (10 + s); };
  auto empty = [&](int s) { return bar0 + 8u * (10 + C::SLOTS + s); };
  volatile uint32_t* tslot = reinterpret_cast<volatile uint32_t*>(smem + C::bar_off + 240);
  volatile int* serr = reinterpret_cast<volatile int*>(smem + C::bar_off + 248);

  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  // the longest rows of a long sequence first
  const int h = blockIdx.x % g.Hq, row0 = (g.units - 1 - blockIdx.x / g.Hq) * C::TILES * TILE;
  // key blocks [first, last) of a tile; blocks are aligned to 128 rows, so the last one of a tile is its diagonal.  They are
  // taken from the diagonal down: the first copies then wait for nothing that has to be looked up.
  auto last_block = [&](int a) { return a < C::TILES && row0 + a * TILE < g.T ? row0 / TILE + a + 1 : 0; };
  const int last0 = last_block(0), last1 = last_block(1), B1 = max(last0, last1), kh = h / g.group;
  if (warp == C::LOAD) {
    if (elect_one()) {
      *serr = 0;
      mbar_init(qfull, 1);
      for (int a = 0; a < 2; ++a) {
        mbar_init(sfull(a), 1);
        mbar_init(sread(a), 4);
        mbar_init(pfull(a), 4);
        mbar_init(pvdone(a), 1);
      }
      mbar_init(drained, 1);
      for (int s = 0; s < C::SLOTS; ++s) {
        mbar_init(full(s), 1);
        mbar_init(empty(s), 1);
      }
      fence_barrier_init();
      mbar_expect_tx(qfull, C::TILES * C::TB);                                     // rows past the end read as zero
      for (int a = 0; a < C::TILES; ++a) load_tile<DH>(base + C::q_off + a * C::TB, &tmQ, qfull, h, row0 + a * TILE);
      for (int i = 0; i < 2; ++i) {
        mbar_expect_tx(full(i), C::TB);
        load_tile<DH>(base + C::ring_off + i * C::TB, i ? &tmV : &tmK, full(i), kh, (B1 - 1) * TILE);
      }
    }
    __syncwarp();
  }
  if (warp == C::ISSUE) tmem_alloc(tslot, C::COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tm = uniform(*tslot);
  // A first row without keys starts at itself: its tile's later rows begin no earlier.
  auto first_block = [&](int a) {
    const int r = row0 + a * TILE;
    return a < C::TILES && r < g.T ? first_key(g.cu, g.nseq, g.window, r) / TILE : 0;
  };
  const int first0 = uniform(first_block(0)), first1 = uniform(first_block(1));
  const int B0 = last1 ? min(first0, first1) : first0;
  const uint32_t tS = tm;
  auto tP = [&](int a) { return tm + C::P_OFF + a * (TILE / 2); };
  auto tO = [&](int a) { return tm + C::O_OFF + a * DH; };

  // 384 threads launch with 168 registers each, 2 x 216 + 72 = 3 x 168; 256 (twice on an SM) with 128, 216 + 40 = 2 x 128
  if (warp >= C::ISSUE) {
    if (C::TILES == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;"); else asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (warp == C::LOAD) {
      // ---------------- TMA loads: K and V of a block in turn ----------------
      const int n = 2 * (B1 - B0);
      int i = 2;                                                    // the first block is on its way
      for (; i < n && !*serr; ++i) {
        const int s = i % C::SLOTS;
        wait(empty(s), ((i / C::SLOTS) & 1) ^ 1, serr);
        if (elect_one()) {
          mbar_expect_tx(full(s), C::TB);
          load_tile<DH>(base + C::ring_off + s * C::TB, (i & 1) ? &tmV : &tmK, full(s), kh, (B1 - 1 - (i >> 1)) * TILE);
        }
      }
      if (*serr) {        // a wait ran out: let the copies in flight land before the CTA ends
        volatile int ignore = 0;
        mbar_wait(qfull, 0, &ignore);
        for (int u = max(0, i - C::SLOTS); u < i; ++u) mbar_wait(full(u % C::SLOTS), (u / C::SLOTS) & 1, &ignore);
      }
    } else if (warp == C::ISSUE) {
      // ---------------- products (the whole warp waits, one lane issues) ----------------
      constexpr uint32_t idS = mma_desc<T>(TILE, TILE, 0, 0), idO = mma_desc<T>(TILE, DH, 0, 1);
      const int begin = max(0, __ldg(g.cu)), end = min(g.T, __ldg(g.cu + g.nseq));
      auto slot_full = [&](int i) { wait(full(i % C::SLOTS), (i / C::SLOTS) & 1, serr); };
      auto scores = [&](int a, int j, bool release) {               // S = Q K_j^T into columns that are free
        const int i = 2 * (B1 - 1 - j), s = i % C::SLOTS;
        slot_full(i);
        tc_fence_after();
        if (elect_one()) {
          const uint64_t q = desc_dims(base + C::q_off + a * C::TB, 0), k = desc_dims(base + C::ring_off + s * C::TB, 0);
#pragma unroll
          for (int u = 0; u < DH / 16; ++u) umma_bf16(tS, q + dims_step(u), k + dims_step(u), idS, u != 0);
          umma_commit(sfull(a));
          if (release) umma_commit(empty(s));
        }
        __syncwarp();
      };
      auto values = [&](int a, int j, int n, bool release) {        // O += P V_j, n-th block of the tile
        const int i = 2 * (B1 - 1 - j) + 1, s = i % C::SLOTS;
        slot_full(i);
        if (j * TILE < begin || (j + 1) * TILE > end) blank_rows<DH>(smem + C::ring_off + s * C::TB, j * TILE, begin, end, lane);
        const uint64_t v = desc_rows(base + C::ring_off + s * C::TB, 0);
        wait(pfull(a), n & 1, serr);
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int u = 0; u < TILE / 16; ++u) umma_ts(tO(a), tP(a) + 8 * u, v + rows_step(u), idO, n > 0 || u != 0);
          if (release) umma_commit(empty(s));
          umma_commit(pvdone(a));
        }
        __syncwarp();
      };
      wait(qfull, 0, serr);
      if (C::TURNS) {
        // one warp for both tiles: S is free once the scores of the turn before have been read
        auto has = [&](int a, int j) { return a ? j >= first1 && j < last1 : j >= first0 && j < last0; };
        int before = -1, phase = 0;                                 // tile of the turn before, and which of its reads
        auto turn = [&](int a, int j) {
          if (before >= 0) wait(sread(before), phase & 1, serr);
          before = a;
          phase = (a ? last1 : last0) - 1 - j;
          scores(a, j, a == 1 || !has(1, j));
        };
        if (has(0, B1 - 1)) turn(0, B1 - 1);
        if (has(1, B1 - 1)) turn(1, B1 - 1);
        for (int j = B1 - 1; j >= B0; --j) {
          if (has(0, j - 1)) turn(0, j - 1);
          if (has(0, j)) values(0, j, last0 - 1 - j, !has(1, j));
          if (has(1, j - 1)) turn(1, j - 1);
          if (has(1, j)) values(1, j, last1 - 1 - j, true);
        }
      } else {
        // the next scores go behind the softmax's read of the last ones
        scores(0, B1 - 1, true);
        for (int j = B1 - 1, n = 0; j >= B0; --j, ++n) {
          if (j > B0) {
            wait(sread(0), n & 1, serr);
            scores(0, j - 1, true);
          }
          values(0, j, n, true);
        }
      }
      drain_products(drained, serr);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    // ---------------- softmax: one row per thread ----------------
    const int a = warp >> 2, b0 = a ? first1 : first0, b1 = a ? last1 : last0;
    const int row = row0 + a * TILE + (warp & 3) * 32 + lane;
    const uint32_t tl = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_addr = tS + tl, o_addr = tO(a) + tl, p_addr = tP(a) + tl;
    const int lo = row < g.T ? first_key(g.cu, g.nseq, g.window, row) : row + 1;
    const int w_lo = __shfl_sync(0xffffffffu, lo, 31), w_row = row - lane;          // lo ascends with the row
    float m = -INFINITY, l = 0.f;
    int n = 0;
    for (int j = b1 - 1; j >= b0; --j, ++n) {
      wait(sfull(a), n & 1, serr);
      tc_fence_after();
      uint32_t x[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld32(s_addr + 32 * c, x[c]);
      tmem_ld_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(sread(a));
      const int k0 = j * TILE;
      const bool mask = k0 < w_lo || k0 + TILE - 1 > w_row;          // some row of this warp hides some key of this block
      if (mask) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const uint32_t seen = range_bits(k0 + 32 * c, lo, row);
#pragma unroll
          for (int i = 0; i < 32; ++i) x[c][i] = seen & (1u << i) ? x[c][i] : 0xff800000u;      // -inf
        }
      }
      float mx[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        mx[c] = __uint_as_float(x[c][0]);
#pragma unroll
        for (int i = 1; i < 31; i += 2) mx[c] = max3_nan(mx[c], __uint_as_float(x[c][i]), __uint_as_float(x[c][i + 1]));
        mx[c] = max_nan(mx[c], __uint_as_float(x[c][31]));
      }
      const float top = max_nan(max_nan(mx[0], mx[1]), max_nan(mx[2], mx[3])) * g.scale_log2;
      // m: the exponent that is subtracted; -inf while the row has seen no key.  A NaN score makes the sum NaN for good.
      const bool grow = !(top <= m + LAG) || (m == -INFINITY && top > -INFINITY);
      const float m_new = grow ? top : m;
      const bool rescale = __any_sync(0xffffffffu, grow && m != -INFINITY);
      if (rescale) {
        wait(pvdone(a), (n - 1) & 1, serr);                          // n > 0: some row has an m
        tc_fence_after();
        const float f = grow ? ex2(m - m_new) : 1.f;                 // m = -inf: 0, and O is still zero
        l = f == 0.f && l == INFINITY ? 0.f : l * f;                 // infinite: weights of a maximum far below (see FAR)
#pragma unroll
        for (int c = 0; c < DH / 32; ++c) {
          uint32_t o[32];
          tmem_ld32(o_addr + 32 * c, o);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
          tmem_st32(o_addr + 32 * c, o);
        }
      }
      m = m_new;
      const float sub = m == -INFINITY ? 0.f : m;
      f32x2 sum = pair(0.f, 0.f);
#pragma unroll
      for (int c = 0; c < 4; ++c) {                                  // 32 keys = 16 columns of packed weights
        uint32_t p[16];
        sum = add2(sum, mask ? weights<T, 0>(x[c], g.scale_log2, sub, p) : weights<T, C::EMU>(x[c], g.scale_log2, sub, p));
        if (c == 0 && n > 0 && !rescale) {                           // the last product has read the last weights
          wait(pvdone(a), (n - 1) & 1, serr);
          tc_fence_after();
        }
        tmem_st16(p_addr + 16 * c, p);
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(pfull(a));
      float s0, s1;
      split(sum, s0, s1);
      l += s0 + s1;
    }
    // ---------------- output ----------------
    const bool some = n > 0;
    if (some) wait(pvdone(a), (n - 1) & 1, serr);
    tc_fence_after();
    // A row whose maximum is infinite is decided here and not by its weights, as the polynomial turns the exponents NaN and -inf
    // into 2^-126: a score of +inf makes the row NaN, and a row that has seen nothing but -inf is a row without keys.  (Such
    // weights beside a finite maximum are at most 2^-118 of the sum.)
    if (m == INFINITY) l = NAN;
    if (m == -INFINITY) l = 0.f;
    const float inv = some && l != 0.f ? 1.f / l : 0.f;             // no key: zero (NaN sums stay NaN)
    T* o_row = out + ((long long)row * g.Hq + h) * g.D;
    float bad[4] = {0.f, 0.f, 0.f, 0.f};                             // one is NaN once an output is not finite
#pragma unroll
    for (int c = 0; c < DH / 32; ++c) {
      uint32_t o[32];
      if (some) {
        tmem_ld32(o_addr + 32 * c, o);
        tmem_ld_wait();
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = 0;
      }
      if (row < g.T) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float f[16];
          uint32_t w[8];
#pragma unroll
          for (int i = 0; i < 16; ++i) f[i] = inv == 0.f ? 0.f : __uint_as_float(o[16 * u + i]) * inv;
#pragma unroll
          for (int i = 0; i < 16; ++i) bad[i & 3] = fmaf(f[i], 0.f, bad[i & 3]);
#pragma unroll
          for (int i = 0; i < 8; ++i) w[i] = Elem<T>::pack(f[2 * i], f[2 * i + 1]);
          store16(o_row, 32 * c + 16 * u, g.D, w);
          if (out_lo) {                                            // what the rounding left
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float2 r = Elem<T>::unpack(w[i]);
              w[i] = Elem<T>::pack(f[2 * i] - r.x, f[2 * i + 1] - r.y);
            }
            store16(out_lo + (o_row - out), 32 * c + 16 * u, g.D, w);
          }
        }
      }
    }
    const float lse2 = inv == 0.f ? -INFINITY : m + log2f(l);
    if (lse && row < g.T) lse[(long long)h * g.T + row] = lse2 * (1.f / LOG2E);
    // outputs that are not finite though the scores are: a value that the row does not see, or weights of a maximum far below
    const bool again = row < g.T && fabsf(m) < INFINITY && l == l && ((bad[0] + bad[1]) + (bad[2] + bad[3]) != 0.f || fabsf(m) > FAR);
    unsigned todo = __ballot_sync(0xffffffffu, again);
    for (; __builtin_expect(todo != 0, 0); todo &= todo - 1) {
      const int who = __ffs(todo) - 1;
      __syncwarp();                                                  // after the lane's own stores
      redo_row<T>(g, out, out_lo, lse, h, w_row + who, __shfl_sync(0xffffffffu, lo, who));
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == C::ISSUE) tmem_dealloc(tm, C::COLS);
  if (threadIdx.x == 0 && *serr) atomicExch(gerr, 1);
}

template <typename T, int DH>
int launch(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, void* o, void* o_lo, float* lse, const Geo& g, int* err,
           cudaStream_t st) {
  auto kern = packed_fwd_kernel<T, DH>;
  static std::atomic<unsigned long long> set{0};
  if (int rc = allow_smem(kern, Cfg<DH>::total, set)) return rc;
  kern<<<(unsigned)(g.Hq * g.units), Cfg<DH>::NT, Cfg<DH>::total, st>>>(mq, mk, mv, (T*)o, (T*)o_lo, lse, g, err);
  DMB_CHECK_LAUNCH();
  return 0;
}

}  // namespace

// q [T, Hq, D] (row stride, head stride), k / v [T, Hkv, D] likewise, 16-bit elements (half: fp16, else bf16); o [T, Hq, D]
// contiguous; o_lo: like o or null, what the rounding of o left (the backward pass forms do . o from both); lse [Hq, T] fp32 or
// null.  Strides are multiples of 8 elements, pointers 16-byte aligned, D a multiple of 8 up to 128 (the caller checks).
extern "C" int dmb_packed_attn_fwd(const void* q, long long q_rs, long long q_hs, const void* k, long long k_rs, long long k_hs,
                                   const void* v, long long v_rs, long long v_hs, const int* cu, int nseq, void* o, void* o_lo,
                                   float* lse, int T, int Hq, int Hkv, int D, int window, float scale, int half, int* err, void* stream) {
  if (T <= 0) return 0;
  if (D <= 0 || D > 128 || (D & 7) || Hkv <= 0 || Hq % Hkv || nseq < 0) return -1;
  CUtensorMap mq, mk, mv;
  int rc = bind_context();
  if (rc == 0) rc = make_map_rows(&mq, q, D, Hq, T, q_rs, q_hs);
  if (rc == 0) rc = make_map_rows(&mk, k, D, Hkv, T, k_rs, k_hs);
  if (rc == 0) rc = make_map_rows(&mv, v, D, Hkv, T, v_rs, v_hs);
  if (rc) return rc;
  const int rows = (D <= 64 ? Cfg<64>::TILES : Cfg<128>::TILES) * TILE, units = (int)(((long long)T + rows - 1) / rows);
  if ((long long)units * Hq > 0x7fffffffLL) return -1;
  const Geo g{cu, nseq, T, Hq, Hq / Hkv, D, window, units, scale * LOG2E, {q, q_rs, q_hs}, {k, k_rs, k_hs}, {v, v_rs, v_hs}};
  cudaStream_t st = (cudaStream_t)stream;
  if (half) return D <= 64 ? launch<__half, 64>(mq, mk, mv, o, o_lo, lse, g, err, st) : launch<__half, 128>(mq, mk, mv, o, o_lo, lse, g, err, st);
  return D <= 64 ? launch<bf16, 64>(mq, mk, mv, o, o_lo, lse, g, err, st) : launch<bf16, 128>(mq, mk, mv, o, o_lo, lse, g, err, st);
}
