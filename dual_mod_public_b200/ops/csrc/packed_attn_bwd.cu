// Backward of the causal attention over packed sequences (packed_attn_fwd.cu), bf16, on the 5th-generation tensor cores.
//
//   p_ij = exp(s_ij - lse_i),  delta_i = do_i . o_i,  ds_ij = p_ij (do_i . v_j - delta_i)
//   dv_j = sum_i p_ij do_i,   dk_j = scale sum_i ds_ij q_i,   dq_i = scale sum_j ds_ij k_j
//
// Two kernels, each owning what it writes, so nothing is accumulated through memory and results do not depend on any order:
//   dkv   a CTA per (key head, 128 keys); streams the query tiles (of all heads of the group) that see the keys.  Scores are
//         formed transposed, S^T = K Q^T and dP^T = V dO^T: a key per lane of tensor memory, so P^T and dS^T are written
//         back there as the A operands of dV += P^T dO and dK += dS^T Q
//   dq    a CTA per (query head, 128 queries); streams the key blocks: S = Q K^T, dP = dO V^T, dQ += dS K
// The price is that S and dP are formed twice (seven products of 128 x 128 x D per tile instead of five); one kernel would
// have to add dQ tiles through memory in whatever order its CTAs run.
//
// Both: warps 0..7 do the elementwise work (warps w and w + 4 share the lanes 32 (w % 4) .. and take half of the columns
// each), warp 8 issues the products, warp 9 loads.  The products of one step are issued in the order in which their operands
// come free, so the tensor pipe works on (dV, next S) while the math warps form dS, and on (dK or dQ, next dP) while they
// form the next P.  P and dS are rounded to bf16 (relative 2^-8 at most, as o was); everything else is fp32.
//
// A first small kernel forms delta and scales lse to base 2 (+inf for rows without keys and for the padding of the last tile,
// which makes their weights zero).
#include "packed.cuh"

using namespace packed;

namespace {

constexpr int NT = 384;

// aux: [2][Hq][Tp] fp32 (lse in base 2, delta), Tp = T rounded up to whole tiles
template <int LANES>
__global__ void __launch_bounds__(256) packed_delta_kernel(const bf16* __restrict__ o, const bf16* __restrict__ go, long long g_rs,
                                                           long long g_hs, const float* __restrict__ lse, float* __restrict__ aux,
                                                           const int* __restrict__ cu, int nseq, int T, int Tp, int Hq, int D) {
  const long long w = ((long long)blockIdx.x * 256 + threadIdx.x) / LANES;      // (row, head), LANES threads of 8 dims each
  const int sub = threadIdx.x % LANES;
  const long long row = w / Hq;
  const int h = (int)(w - row * Hq);
  if (row >= Tp) return;                                                        // whole groups leave together
  float s = 0.f;
  const bool inside = row < T && row >= __ldg(cu) && row < __ldg(cu + nseq);    // padding rows may hold anything
  if (inside && sub * 8 < D) {
    const uint4 a = *reinterpret_cast<const uint4*>(o + (row * Hq + h) * D + sub * 8);
    const uint4 b = *reinterpret_cast<const uint4*>(go + row * g_rs + h * g_hs + sub * 8);
    const uint32_t x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 p = unpack_bf16(x[i]), q = unpack_bf16(y[i]);
      s = fmaf(p.x, q.x, s);
      s = fmaf(p.y, q.y, s);
    }
  }
#pragma unroll
  for (int i = LANES / 2; i > 0; i >>= 1) s += __shfl_xor_sync(0xffffffffu, s, i);
  if (sub == 0) {
    const float L = inside ? lse[(long long)h * T + row] : -INFINITY;
    aux[(long long)h * Tp + row] = L == -INFINITY ? INFINITY : L * LOG2E;
    aux[((long long)Hq + h) * Tp + row] = s;
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
  static constexpr int TB = TILE * DH * 2;
  static constexpr int ST = DH == 128 ? 2 : 4;             // ring stages, two tiles each
  static constexpr int own_off = 0, ring_off = 2 * TB;     // the owner's two tiles, then the ring
  static constexpr int aux_off = ring_off + ST * 2 * TB;   // dkv: per stage 128 lse and 128 delta
  static constexpr int bar_off = aux_off + ST * 1024;
  static constexpr int total = bar_off + 256;
};

// ---------------------------------------------------------------------------------------------------------------------------
template <int DH>
__global__ void __launch_bounds__(NT, 1) packed_dkv_kernel(
    const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
    const __grid_constant__ CUtensorMap tmG, bf16* __restrict__ dk, bf16* __restrict__ dv, const Geo g, int* __restrict__ gerr) {
  using C = Cfg<DH>;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t base = smem_u32(smem);
  if (base & 1023u) {
    if (threadIdx.x == 0) atomicExch(gerr, 2);
    return;
  }
  const uint32_t bar0 = base + C::bar_off;
  // barriers: own, sfull, dpfull, pfull, dsfull, done, drained, qfull[ST], gfull[ST], empty[ST]
  const uint32_t own = bar0, sfull = bar0 + 8, dpfull = bar0 + 16, pfull = bar0 + 24, dsfull = bar0 + 32, done = bar0 + 40,
                 drained = bar0 + 48;
  auto qfull = [&](int s) { return bar0 + 56 + 8u * s; };
  auto gfull = [&](int s) { return bar0 + 56 + 8u * (C::ST + s); };
  auto empty = [&](int s) { return bar0 + 56 + 8u * (2 * C::ST + s); };
  volatile uint32_t* tslot = reinterpret_cast<volatile uint32_t*>(smem + C::bar_off + 240);
  volatile int* serr = reinterpret_cast<volatile int*>(smem + C::bar_off + 248);
  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  // the first keys of a long sequence are seen by the most queries: they come first
  const int kh = blockIdx.x % g.Hkv, kt = blockIdx.x / g.Hkv, key0 = kt * TILE;
  const int last = last_query(g.cu, g.nseq, g.window, g.T, min(g.T, key0 + TILE) - 1);
  const int nq = uniform(max(kt, last / TILE)) - kt + 1, n_it = nq * g.group;         // query tiles kt .. kt + nq - 1 of each head

  if (threadIdx.x == 0) {
    *serr = 0;
    mbar_init(own, 1);
    mbar_init(sfull, 1);
    mbar_init(dpfull, 1);
    mbar_init(pfull, 8);
    mbar_init(dsfull, 8);
    mbar_init(done, 1);
    mbar_init(drained, 1);
    for (int s = 0; s < C::ST; ++s) {
      mbar_init(qfull(s), 1);
      mbar_init(gfull(s), 1);
      mbar_init(empty(s), 1);
    }
    fence_barrier_init();
  }
  if (warp == 8) tmem_alloc(tslot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tm = uniform(*tslot);
  const uint32_t tS = tm, tdP = tm + TILE, tdV = tm + 2 * TILE, tdK = tdV + DH;
  const uint32_t sK = base + C::own_off, sV = sK + C::TB;
  auto sQ = [&](int s) { return base + C::ring_off + s * 2 * C::TB; };
  auto sG = [&](int s) { return sQ(s) + C::TB; };

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");          // 2 x 216 + 72 = 3 x 168
    if (warp == 9) {
      if (elect_one()) {
        mbar_expect_tx(own, 2 * C::TB);
        load_tile<DH>(sK, &tmK, own, kh, key0);
        load_tile<DH>(sV, &tmV, own, kh, key0);
      }
      int i = 0, qi = 0, h = kh * g.group;
      for (; i < n_it && !*serr; ++i) {
        const int s = i % C::ST, q0 = (kt + qi) * TILE;
        const float* ax = g.aux + (long long)h * g.Tp + q0;
        const uint32_t sa = base + C::aux_off + s * 1024;
        wait(empty(s), ((i / C::ST) & 1) ^ 1, serr);
        if (elect_one()) {
          mbar_expect_tx(qfull(s), C::TB + 512);
          load_tile<DH>(sQ(s), &tmQ, qfull(s), h, q0);
          load_bulk(sa, ax, 512, qfull(s));
          mbar_expect_tx(gfull(s), C::TB + 512);
          load_tile<DH>(sG(s), &tmG, gfull(s), h, q0);
          load_bulk(sa + 512, ax + (long long)g.Hq * g.Tp, 512, gfull(s));
        }
        if (++qi == nq) { qi = 0; ++h; }
      }
      if (*serr) {          // a wait ran out: let the copies in flight land before the CTA ends
        volatile int ignore = 0;
        mbar_wait(own, 0, &ignore);
        for (int u = max(0, i - C::ST); u < i; ++u) {
          mbar_wait(qfull(u % C::ST), (u / C::ST) & 1, &ignore);
          mbar_wait(gfull(u % C::ST), (u / C::ST) & 1, &ignore);
        }
      }
    } else if (warp == 8) {
      constexpr uint32_t idS = mma_desc<bf16>(TILE, TILE, 0, 0), idG = mma_desc<bf16>(TILE, DH, 0, 1);
      const int begin = max(0, __ldg(g.cu)), end = min(g.T, __ldg(g.cu + g.nseq));
      auto padded = [&](int q0) { return q0 < begin || q0 + TILE > end; };
      auto scores = [&](int i, int q0) {                 // S^T = K Q_i^T
        const int s = i % C::ST;
        wait(qfull(s), (i / C::ST) & 1, serr);
        if (padded(q0)) blank_rows<DH>(smem + C::ring_off + s * 2 * C::TB, q0, begin, end, lane);
        tc_fence_after();
        if (elect_one()) {
          const uint64_t k = desc_dims(sK, 0), q = desc_dims(sQ(s), 0);
#pragma unroll
          for (int u = 0; u < DH / 16; ++u) umma_bf16(tS, k + dims_step(u), q + dims_step(u), idS, u != 0);
          umma_commit(sfull);
        }
        __syncwarp();
      };
      auto dscores = [&](int i, int q0) {                // dP^T = V dO_i^T
        const int s = i % C::ST;
        wait(gfull(s), (i / C::ST) & 1, serr);
        if (padded(q0)) blank_rows<DH>(smem + C::ring_off + s * 2 * C::TB + C::TB, q0, begin, end, lane);
        tc_fence_after();
        if (elect_one()) {
          const uint64_t v = desc_dims(sV, 0), go = desc_dims(sG(s), 0);
#pragma unroll
          for (int u = 0; u < DH / 16; ++u) umma_bf16(tdP, v + dims_step(u), go + dims_step(u), idS, u != 0);
          umma_commit(dpfull);
        }
        __syncwarp();
      };
      wait(own, 0, serr);
      scores(0, key0);
      dscores(0, key0);
      int qi = 0;
      for (int i = 0; i < n_it; ++i) {
        const int s = i % C::ST;
        if (++qi == nq) qi = 0;                          // of the next step
        wait(pfull, i & 1, serr);
        tc_fence_after();
        if (elect_one()) {
          const uint64_t go = desc_rows(sG(s), 0);
#pragma unroll
          for (int u = 0; u < TILE / 16; ++u)            // the halves of P^T lie behind each other's scores: 0 .. 31 and 64 .. 95
            umma_ts(tdV, tS + (u / 4) * 64 + (u % 4) * 8, go + rows_step(u), idG, i > 0 || u != 0);
        }
        __syncwarp();
        if (i + 1 < n_it) scores(i + 1, key0 + qi * TILE);
        wait(dsfull, i & 1, serr);
        tc_fence_after();
        if (elect_one()) {
          const uint64_t q = desc_rows(sQ(s), 0);
#pragma unroll
          for (int u = 0; u < TILE / 16; ++u)
            umma_ts(tdK, tdP + (u / 4) * 64 + (u % 4) * 8, q + rows_step(u), idG, i > 0 || u != 0);
          umma_commit(empty(s));
          if (i + 1 == n_it) umma_commit(done);
        }
        __syncwarp();
        if (i + 1 < n_it) dscores(i + 1, key0 + qi * TILE);
      }
      drain_products(drained, serr);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int half = warp >> 2, key = key0 + (warp & 3) * 32 + lane;
    const uint32_t tl = (uint32_t)((warp & 3) * 32) << 16;
    const int hi = key < g.T ? last_query(g.cu, g.nseq, g.window, g.T, key) : key - 1;
    const int w_hi = __shfl_sync(0xffffffffu, hi, 0), w_key = key - lane + 31;        // hi ascends with the key
    int qi = 0;
    for (int i = 0; i < n_it; ++i) {
      const int s = i % C::ST, q0 = (kt + qi) * TILE + half * 64;
      if (++qi == nq) qi = 0;
      const float4* lse = reinterpret_cast<const float4*>(smem + C::aux_off + s * 1024) + half * 16;
      const float4* delta = lse + 32;
      wait(sfull, i & 1, serr);
      wait(qfull(s), (i / C::ST) & 1, serr);               // lse arrived with the queries
      tc_fence_after();
      uint32_t x[2][32];
      tmem_ld32(tS + tl + half * 64, x[0]);
      tmem_ld32(tS + tl + half * 64 + 32, x[1]);
      tmem_ld_wait();
      float p[64];
#pragma unroll
      for (int c = 0; c < 16; ++c) {
        const float4 L = lse[c];
        p[4 * c] = exp2f(fmaf(__uint_as_float(x[c >> 3][(4 * c) & 31]), g.scale_log2, -L.x));
        p[4 * c + 1] = exp2f(fmaf(__uint_as_float(x[c >> 3][(4 * c + 1) & 31]), g.scale_log2, -L.y));
        p[4 * c + 2] = exp2f(fmaf(__uint_as_float(x[c >> 3][(4 * c + 2) & 31]), g.scale_log2, -L.z));
        p[4 * c + 3] = exp2f(fmaf(__uint_as_float(x[c >> 3][(4 * c + 3) & 31]), g.scale_log2, -L.w));
      }
      const bool mask = q0 < w_key || q0 + 63 > w_hi;
      const int c_lo = key - q0, c_hi = hi - q0;
      if (mask) {
#pragma unroll
        for (int c = 0; c < 64; ++c)
          if (c < c_lo || c > c_hi) p[c] = 0.f;
      }
      {
        uint32_t w[32];
#pragma unroll
        for (int c = 0; c < 32; ++c) w[c] = pack_bf16(p[2 * c], p[2 * c + 1]);
        tmem_st32(tS + tl + half * 64, w);
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(pfull);
      wait(dpfull, i & 1, serr);
      wait(gfull(s), (i / C::ST) & 1, serr);
      tc_fence_after();
      tmem_ld32(tdP + tl + half * 64, x[0]);
      tmem_ld32(tdP + tl + half * 64 + 32, x[1]);
      tmem_ld_wait();
#pragma unroll
      for (int c = 0; c < 16; ++c) {
        const float4 d = delta[c];
        p[4 * c] *= __uint_as_float(x[c >> 3][(4 * c) & 31]) - d.x;
        p[4 * c + 1] *= __uint_as_float(x[c >> 3][(4 * c + 1) & 31]) - d.y;
        p[4 * c + 2] *= __uint_as_float(x[c >> 3][(4 * c + 2) & 31]) - d.z;
        p[4 * c + 3] *= __uint_as_float(x[c >> 3][(4 * c + 3) & 31]) - d.w;
      }
      if (mask) {                                          // 0 x (what a padding row's product left) is not zero
#pragma unroll
        for (int c = 0; c < 64; ++c)
          if (c < c_lo || c > c_hi) p[c] = 0.f;
      }
      {
        uint32_t w[32];
#pragma unroll
        for (int c = 0; c < 32; ++c) w[c] = pack_bf16(p[2 * c], p[2 * c + 1]);
        tmem_st32(tdP + tl + half * 64, w);
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(dsfull);
    }
    wait(done, 0, serr);
    tc_fence_after();
    const long long off = ((long long)key * g.Hkv + kh) * g.D;
    if (half == 0) store_row<DH>(tdV + tl, dv + off, g.D, 1.f, key < g.T);
    else store_row<DH>(tdK + tl, dk + off, g.D, g.scale, key < g.T);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 8) tmem_dealloc(tm, 512);
  if (threadIdx.x == 0 && *serr) atomicExch(gerr, 1);
}

// ---------------------------------------------------------------------------------------------------------------------------
template <int DH>
__global__ void __launch_bounds__(NT, 1) packed_dq_kernel(
    const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
    const __grid_constant__ CUtensorMap tmG, bf16* __restrict__ dq, const Geo g, int* __restrict__ gerr) {
  using C = Cfg<DH>;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t base = smem_u32(smem);
  if (base & 1023u) {
    if (threadIdx.x == 0) atomicExch(gerr, 2);
    return;
  }
  const uint32_t bar0 = base + C::bar_off;
  // barriers: own, sfull, dpfull, sread, dsfull, done, drained, kfull[ST], vfull[ST], empty[ST]
  const uint32_t own = bar0, sfull = bar0 + 8, dpfull = bar0 + 16, sread = bar0 + 24, dsfull = bar0 + 32, done = bar0 + 40,
                 drained = bar0 + 48;
  auto kfull = [&](int s) { return bar0 + 56 + 8u * s; };
  auto vfull = [&](int s) { return bar0 + 56 + 8u * (C::ST + s); };
  auto empty = [&](int s) { return bar0 + 56 + 8u * (2 * C::ST + s); };
  volatile uint32_t* tslot = reinterpret_cast<volatile uint32_t*>(smem + C::bar_off + 240);
  volatile int* serr = reinterpret_cast<volatile int*>(smem + C::bar_off + 248);
  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int h = blockIdx.x % g.Hq, qt = g.tiles - 1 - blockIdx.x / g.Hq, row0 = qt * TILE;
  const int kb0 = uniform(min(qt, first_key(g.cu, g.nseq, g.window, row0) / TILE)), n_it = qt - kb0 + 1;

  if (threadIdx.x == 0) {
    *serr = 0;
    mbar_init(own, 1);
    mbar_init(sfull, 1);
    mbar_init(dpfull, 1);
    mbar_init(sread, 8);
    mbar_init(dsfull, 8);
    mbar_init(done, 1);
    mbar_init(drained, 1);
    for (int s = 0; s < C::ST; ++s) {
      mbar_init(kfull(s), 1);
      mbar_init(vfull(s), 1);
      mbar_init(empty(s), 1);
    }
    fence_barrier_init();
  }
  if (warp == 8) tmem_alloc(tslot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tm = uniform(*tslot);
  const uint32_t tS = tm, tdP = tm + TILE, tdQ = tm + 2 * TILE;
  const uint32_t sQ = base + C::own_off, sG = sQ + C::TB;
  auto sK = [&](int s) { return base + C::ring_off + s * 2 * C::TB; };
  auto sV = [&](int s) { return sK(s) + C::TB; };

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == 9) {
      const int kh = h / g.group;
      if (elect_one()) {
        mbar_expect_tx(own, 2 * C::TB);
        load_tile<DH>(sQ, &tmQ, own, h, row0);
        load_tile<DH>(sG, &tmG, own, h, row0);
      }
      int i = 0;
      for (; i < n_it && !*serr; ++i) {
        const int s = i % C::ST, k0 = (kb0 + i) * TILE;
        wait(empty(s), ((i / C::ST) & 1) ^ 1, serr);
        if (elect_one()) {
          mbar_expect_tx(kfull(s), C::TB);
          load_tile<DH>(sK(s), &tmK, kfull(s), kh, k0);
          mbar_expect_tx(vfull(s), C::TB);
          load_tile<DH>(sV(s), &tmV, vfull(s), kh, k0);
        }
      }
      if (*serr) {
        volatile int ignore = 0;
        mbar_wait(own, 0, &ignore);
        for (int u = max(0, i - C::ST); u < i; ++u) {
          mbar_wait(kfull(u % C::ST), (u / C::ST) & 1, &ignore);
          mbar_wait(vfull(u % C::ST), (u / C::ST) & 1, &ignore);
        }
      }
    } else if (warp == 8) {
      constexpr uint32_t idS = mma_desc<bf16>(TILE, TILE, 0, 0), idG = mma_desc<bf16>(TILE, DH, 0, 1);
      const int begin = max(0, __ldg(g.cu)), end = min(g.T, __ldg(g.cu + g.nseq));
      auto scores = [&](int i) {                         // S = Q K_i^T
        const int s = i % C::ST, k0 = (kb0 + i) * TILE;
        wait(kfull(s), (i / C::ST) & 1, serr);
        if (k0 < begin || k0 + TILE > end) blank_rows<DH>(smem + C::ring_off + s * 2 * C::TB, k0, begin, end, lane);
        tc_fence_after();
        if (elect_one()) {
          const uint64_t q = desc_dims(sQ, 0), k = desc_dims(sK(s), 0);
#pragma unroll
          for (int u = 0; u < DH / 16; ++u) umma_bf16(tS, q + dims_step(u), k + dims_step(u), idS, u != 0);
          umma_commit(sfull);
        }
        __syncwarp();
      };
      auto dscores = [&](int i) {                        // dP = dO V_i^T
        const int s = i % C::ST;
        wait(vfull(s), (i / C::ST) & 1, serr);
        tc_fence_after();
        if (elect_one()) {
          const uint64_t go = desc_dims(sG, 0), v = desc_dims(sV(s), 0);
#pragma unroll
          for (int u = 0; u < DH / 16; ++u) umma_bf16(tdP, go + dims_step(u), v + dims_step(u), idS, u != 0);
          umma_commit(dpfull);
        }
        __syncwarp();
      };
      wait(own, 0, serr);
      scores(0);
      dscores(0);
      for (int i = 0; i < n_it; ++i) {
        const int s = i % C::ST;
        if (i + 1 < n_it) {
          wait(sread, i & 1, serr);
          scores(i + 1);
        }
        wait(dsfull, i & 1, serr);
        tc_fence_after();
        if (elect_one()) {
          const uint64_t k = desc_rows(sK(s), 0);
#pragma unroll
          for (int u = 0; u < TILE / 16; ++u)
            umma_ts(tdQ, tdP + (u / 4) * 64 + (u % 4) * 8, k + rows_step(u), idG, i > 0 || u != 0);
          umma_commit(empty(s));
          if (i + 1 == n_it) umma_commit(done);
        }
        __syncwarp();
        if (i + 1 < n_it) dscores(i + 1);
      }
      drain_products(drained, serr);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int half = warp >> 2, row = row0 + (warp & 3) * 32 + lane;
    const uint32_t tl = (uint32_t)((warp & 3) * 32) << 16;
    const int lo = row < g.T ? first_key(g.cu, g.nseq, g.window, row) : row + 1;
    const int w_lo = __shfl_sync(0xffffffffu, lo, 31), w_row = row - lane;
    const float L = g.aux[(long long)h * g.Tp + row], delta = g.aux[((long long)g.Hq + h) * g.Tp + row];
    for (int i = 0; i < n_it; ++i) {
      const int k0 = (kb0 + i) * TILE + half * 64;
      wait(sfull, i & 1, serr);
      tc_fence_after();
      uint32_t x[2][32];
      tmem_ld32(tS + tl + half * 64, x[0]);
      tmem_ld32(tS + tl + half * 64 + 32, x[1]);
      tmem_ld_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(sread);
      float p[64];
#pragma unroll
      for (int c = 0; c < 64; ++c) p[c] = exp2f(fmaf(__uint_as_float(x[c >> 5][c & 31]), g.scale_log2, -L));
      wait(dpfull, i & 1, serr);
      tc_fence_after();
      tmem_ld32(tdP + tl + half * 64, x[0]);
      tmem_ld32(tdP + tl + half * 64 + 32, x[1]);
      tmem_ld_wait();
#pragma unroll
      for (int c = 0; c < 64; ++c) p[c] *= __uint_as_float(x[c >> 5][c & 31]) - delta;
      if (k0 < w_lo || k0 + 63 > w_row) {
        const int c_lo = lo - k0, c_hi = row - k0;
#pragma unroll
        for (int c = 0; c < 64; ++c)
          if (c < c_lo || c > c_hi) p[c] = 0.f;
      }
      {
        uint32_t w[32];
#pragma unroll
        for (int c = 0; c < 32; ++c) w[c] = pack_bf16(p[2 * c], p[2 * c + 1]);
        tmem_st32(tdP + tl + half * 64, w);
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(dsfull);
    }
    wait(done, 0, serr);
    tc_fence_after();
    if (half == 0) store_row<DH>(tdQ + tl, dq + ((long long)row * g.Hq + h) * g.D, g.D, g.scale, row < g.T);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 8) tmem_dealloc(tm, 512);
  if (threadIdx.x == 0 && *serr) atomicExch(gerr, 1);
}

template <int DH>
int launch(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const CUtensorMap& mg, bf16* dq, bf16* dk, bf16* dv,
           const Geo& g, int* err, cudaStream_t st) {
  cudaError_t e = cudaFuncSetAttribute(packed_dkv_kernel<DH>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<DH>::total);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(packed_dq_kernel<DH>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<DH>::total);
  if (e != cudaSuccess) return (int)e;
  packed_dkv_kernel<DH><<<(unsigned)(g.tiles * g.Hkv), NT, Cfg<DH>::total, st>>>(mq, mk, mv, mg, dk, dv, g, err);
  DMB_CHECK_LAUNCH();
  packed_dq_kernel<DH><<<(unsigned)(g.tiles * g.Hq), NT, Cfg<DH>::total, st>>>(mq, mk, mv, mg, dq, g, err);
  DMB_CHECK_LAUNCH();
  return 0;
}

}  // namespace

// bf16: go (gradient of o) [T, Hq, D] and q, k, v by strides as in dmb_packed_attn_fwd; o, dq [T, Hq, D], dk, dv [T, Hkv, D]
// contiguous; lse [Hq, T]; aux fp32 [2, Hq, Tp] with Tp = T rounded up to a multiple of 128.  All gradient rows are written.
extern "C" int dmb_packed_attn_bwd(const void* go, long long g_rs, long long g_hs, const void* q, long long q_rs, long long q_hs,
                                   const void* k, long long k_rs, long long k_hs, const void* v, long long v_rs, long long v_hs,
                                   const void* o, const float* lse, const int* cu, int nseq, float* aux, void* dq, void* dk,
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
  if ((long long)tiles * Hq > 0x7fffffffLL) return -1;
  const Geo g{cu, aux, nseq, T, tiles * TILE, Hq, Hkv, Hq / Hkv, D, window, tiles, scale, scale * LOG2E};
  cudaStream_t st = (cudaStream_t)stream;
  const long long rows = (long long)g.Tp * Hq;
  if (D <= 64) {
    packed_delta_kernel<8><<<(unsigned)((rows * 8 + 255) / 256), 256, 0, st>>>((const bf16*)o, (const bf16*)go, g_rs, g_hs, lse, aux,
                                                                                cu, nseq, T, g.Tp, Hq, D);
  } else {
    packed_delta_kernel<16><<<(unsigned)((rows * 16 + 255) / 256), 256, 0, st>>>((const bf16*)o, (const bf16*)go, g_rs, g_hs, lse, aux,
                                                                                  cu, nseq, T, g.Tp, Hq, D);
  }
  DMB_CHECK_LAUNCH();
  return D <= 64 ? launch<64>(mq, mk, mv, mg, (bf16*)dq, (bf16*)dk, (bf16*)dv, g, err, st)
                 : launch<128>(mq, mk, mv, mg, (bf16*)dq, (bf16*)dk, (bf16*)dv, g, err, st);
}
