// Causal attention over packed sequences, forward, on the 5th-generation tensor cores.
//
//   s_ij = scale q_i . k_j   for first_key(i) <= j <= i,   o_i = sum_j softmax(s_i)_j v_j,   lse_i = log sum_j exp s_ij
//
// q [T, Hq, D], k / v [T, Hkv, D], sequences packed one behind the other on the row axis (packed.cuh); query head h reads key
// head h / (Hq / Hkv).  A tile is 128 consecutive packed rows whatever sequences they belong to, so short sequences cost no
// padding: the keys a tile needs are one contiguous range, and each row masks to its own part of it.
//
// One CTA per (head, pair of query tiles), 256 rows; key blocks of 128 stream through a shared-memory ring and serve both:
//   warps 0..3   softmax of tile 0: every thread owns one row = one lane of tensor memory
//   warps 4..7   softmax of tile 1
//   warp 8       issues S_a = Q_a K^T and O_a += P_a V; P comes from tensor memory, where it overwrites the scores it is
//                made from, so the scores of a tile's next block are issued right behind the product that reads P.  While
//                one tile's softmax runs, the tensor pipe works for the other
//   warp 9       TMA loads
// The running maximum is allowed to lag by up to 8 octaves (P <= 256, exact in the fp32 accumulator's range and no loss of
// relative precision in 16 bits): O is rescaled in tensor memory only when a row's maximum outgrows that, which after the
// first blocks is rare.  Sums are fp32; P is rounded to the operand type, half an ulp per weight (2^-9 relative for bf16).
//
// Every mbarrier wait is bounded in time; on expiry the kernel raises a flag in global memory, stops waiting, lets its own
// copies land (bounded) and releases its tensor memory.
#include "packed.cuh"

using namespace packed;

namespace {

constexpr int NT = 384;              // two softmax warpgroups, one for loads and MMA issue (two of its warps idle)
constexpr float LAG = 8.f;              // octaves

template <int DH>
struct Cfg {
  static constexpr int TB = TILE * DH * 2;                 // one tile
  static constexpr int SLOTS = DH == 128 ? 5 : 8;
  static constexpr int q_off = 0, ring_off = 2 * TB;
  static constexpr int bar_off = ring_off + SLOTS * TB;
  static constexpr int total = bar_off + 256;
};

struct Geo {
  const int* cu;
  int nseq, T, Hq, group, D, window, pairs;
  float scale_log2;
};

template <typename T, int DH>
__global__ void __launch_bounds__(NT, 1) packed_fwd_kernel(
    const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
    T* __restrict__ out, float* __restrict__ lse, const Geo g, int* __restrict__ gerr) {
  using C = Cfg<DH>;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t base = smem_u32(smem);
  if (base & 1023u) {
    if (threadIdx.x == 0) atomicExch(gerr, 2);
    return;
  }
  const uint32_t bar0 = base + C::bar_off;
  // barriers: qfull, sfull[2], pfull[2], ofull[2], full[SLOTS], empty[SLOTS]
  const uint32_t qfull = bar0;
  auto sfull = [&](int a) { return bar0 + 8u * (1 + a); };
  auto pfull = [&](int a) { return bar0 + 8u * (3 + a); };
  auto ofull = [&](int a) { return bar0 + 8u * (5 + a); };
  auto full = [&](int s) { return bar0 + 8u * (7 + s); };
  auto empty = [&](int s) { return bar0 + 8u * (7 + C::SLOTS + s); };
  volatile uint32_t* tslot = reinterpret_cast<volatile uint32_t*>(smem + C::bar_off + 8 * 23);
  volatile int* serr = reinterpret_cast<volatile int*>(smem + C::bar_off + 8 * 24);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // the longest rows of a long sequence first
  const int h = blockIdx.x % g.Hq, pair = g.pairs - 1 - blockIdx.x / g.Hq;
  const int row0 = pair * 2 * TILE;
  // key blocks [b0[a], b1[a]) of each tile; blocks are aligned to 128 rows, so the last one of a tile is its diagonal
  int b0[2], b1[2];
#pragma unroll
  for (int a = 0; a < 2; ++a) {
    const int r = row0 + a * TILE;
    b0[a] = b1[a] = 0;
    if (r < g.T) {
      b1[a] = r / TILE + 1;
      b0[a] = min(first_key(g.cu, g.nseq, g.window, r) / TILE, b1[a]);
      // a first row without keys starts at itself: its tile's later rows begin no earlier
    }
  }
  const int B0 = b1[0] == b0[0] ? b0[1] : (b1[1] == b0[1] ? b0[0] : min(b0[0], b0[1])), B1 = max(b1[0], b1[1]);

  if (threadIdx.x == 0) {
    *serr = 0;
    mbar_init(qfull, 1);
    for (int a = 0; a < 2; ++a) {
      mbar_init(sfull(a), 1);
      mbar_init(pfull(a), 4);
      mbar_init(ofull(a), 1);
    }
    for (int s = 0; s < C::SLOTS; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    fence_barrier_init();
  }
  if (warp == 8) tmem_alloc(tslot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tm = *tslot;
  auto tS = [&](int a) { return tm + a * TILE; };
  auto tO = [&](int a) { return tm + 2 * TILE + a * DH; };

  // 384 threads launch with 168 registers each; 2 x 216 + 72 = 3 x 168
  if (warp >= 8) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
  if (warp == 9) {
    // ---------------- TMA loads: K and V of a block in turn ----------------
    if (lane == 0 && B1 > B0) {
      mbar_expect_tx(qfull, 2 * C::TB);
      load_tile<DH>(base + C::q_off, &tmQ, qfull, h, row0);
      load_tile<DH>(base + C::q_off + C::TB, &tmQ, qfull, h, row0 + TILE);     // rows past the end read as zero
      const int kh = h / g.group, n = 2 * (B1 - B0);
      int i = 0;
      for (; i < n; ++i) {
        const int s = i % C::SLOTS;
        if (!wait_quick(empty(s), ((i / C::SLOTS) & 1) ^ 1, serr)) break;
        mbar_expect_tx(full(s), C::TB);
        load_tile<DH>(base + C::ring_off + s * C::TB, (i & 1) ? &tmV : &tmK, full(s), kh, (B0 + (i >> 1)) * TILE);
      }
      if (*serr) {      // a role gave up: let the copies in flight land before the CTA ends
        volatile int ignore = 0;
        mbar_wait(qfull, 0, &ignore);
        for (int u = max(0, i - C::SLOTS); u < i; ++u) mbar_wait(full(u % C::SLOTS), (u / C::SLOTS) & 1, &ignore);
      }
    }
  } else if (warp == 8) {
    // ---------------- MMA issue (the whole warp waits, one lane issues) ----------------
    constexpr uint32_t idS = mma_desc<T>(TILE, TILE, 0, 0), idO = mma_desc<T>(TILE, DH, 0, 1);
    const int begin = max(0, __ldg(g.cu)), end = min(g.T, __ldg(g.cu + g.nseq));
    auto issue_S = [&](int a, int slot) {
      if (lane == 0) {
        const uint32_t q = base + C::q_off + a * C::TB, k = base + C::ring_off + slot * C::TB;
#pragma unroll
        for (int s = 0; s < DH / 16; ++s) umma_bf16(tS(a), desc_dims(q, s), desc_dims(k, s), idS, s != 0);
        umma_commit(sfull(a));
      }
    };
    bool alive = B1 > B0 && wait_warp(qfull, 0, serr) && wait_warp(full(0), 0, serr);
    int np[2] = {0, 0};                 // P tiles taken, per tile
    if (alive) {
      tc_fence_after();
#pragma unroll
      for (int a = 0; a < 2; ++a)
        if (b0[a] <= B0 && B0 < b1[a]) issue_S(a, 0);
      if (lane == 0) umma_commit(empty(0));
    }
    for (int j = B0; j < B1 && alive; ++j) {
      const int iv = 2 * (j - B0) + 1, sv = iv % C::SLOTS;          // ring positions of V_j and K_{j+1}
      const int ik = iv + 1, sk = ik % C::SLOTS;
      const bool more = j + 1 < B1;
      if (!wait_warp(full(sv), (iv / C::SLOTS) & 1, serr)) { alive = false; break; }
      if (j * TILE < begin || (j + 1) * TILE > end) blank_rows<DH>(smem + C::ring_off + sv * C::TB, j * TILE, begin, end, lane);
      bool k_here = false;
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        if (j >= b0[a] && j < b1[a]) {
          if (!wait_warp(pfull(a), np[a] & 1, serr)) { alive = false; break; }
          ++np[a];
          tc_fence_after();
          if (lane == 0) {
            const uint32_t v = base + C::ring_off + sv * C::TB;
#pragma unroll
            for (int s = 0; s < TILE / 16; ++s) umma_ts(tO(a), tS(a) + 8 * s, desc_rows(v, s), idO, j > b0[a] || s != 0);
            if (j + 1 == b1[a]) umma_commit(ofull(a));
          }
        }
        if (more && j + 1 >= b0[a] && j + 1 < b1[a]) {
          if (!k_here) {
            if (!wait_warp(full(sk), (ik / C::SLOTS) & 1, serr)) { alive = false; break; }
            k_here = true;
            tc_fence_after();
          }
          issue_S(a, sk);
        }
      }
      if (alive && lane == 0) {
        umma_commit(empty(sv));
        if (more) umma_commit(empty(sk));
      }
    }
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    // ---------------- softmax: one row per thread ----------------
    const int a = warp >> 2, r = (warp & 3) * 32 + lane;
    const int row = row0 + a * TILE + r;
    const uint32_t tl = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_addr = tS(a) + tl, o_addr = tO(a) + tl;
    const int lo = row < g.T ? first_key(g.cu, g.nseq, g.window, row) : row + 1;
    const int tile_lo = __shfl_sync(0xffffffffu, lo, 31);          // lo ascends: the last row's is the warp's greatest
    const int w_row0 = row - lane;
    float m = -INFINITY, l = 0.f;
    bool alive = true;
    int n = 0;
    for (int j = b0[a]; j < b1[a]; ++j, ++n) {
      if (!wait_warp(sfull(a), n & 1, serr)) { alive = false; break; }
      tc_fence_after();
      uint32_t x[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld32(s_addr + 32 * c, x[c]);
      tmem_ld_wait();
      const int k0 = j * TILE;
      if (k0 < tile_lo || k0 + TILE - 1 > w_row0) {                // some row of this warp masks some key of this block
        const int c_lo = lo - k0, c_hi = row - k0;
#pragma unroll
        for (int c = 0; c < 128; ++c)
          if (c < c_lo || c > c_hi) x[c >> 5][c & 31] = 0xff800000u;            // -inf
      }
      float mx[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        mx[c] = __uint_as_float(x[c][0]);
#pragma unroll
        for (int i = 1; i < 32; ++i) mx[c] = fmaxf(mx[c], __uint_as_float(x[c][i]));
      }
      const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * g.scale_log2;
      // m: the exponent that is subtracted; -inf while the row has seen no key
      const bool grow = top > m + LAG || (m == -INFINITY && top > -INFINITY);
      const float m_new = grow ? top : m;
      if (__any_sync(0xffffffffu, grow && l > 0.f)) {
        const float f = grow ? exp2f(m - m_new) : 1.f;             // m = -inf: exp2(-inf) = 0, and O is still zero
        l *= f;
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
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < 2; ++c) {                                 // 64 keys = 32 columns of packed weights
        uint32_t p[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const float p0 = exp2f(fmaf(__uint_as_float(x[2 * c + (i >> 4)][2 * (i & 15)]), g.scale_log2, -sub));
          const float p1 = exp2f(fmaf(__uint_as_float(x[2 * c + (i >> 4)][2 * (i & 15) + 1]), g.scale_log2, -sub));
          sum[i & 1] += p0;
          sum[2 + (i & 1)] += p1;
          p[i] = Elem<T>::pack(p0, p1);
        }
        tmem_st32(s_addr + 32 * c, p);
      }
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(pfull(a));
    }
    // ---------------- output ----------------
    const bool some = alive && b1[a] > b0[a] && wait_warp(ofull(a), 0, serr);
    tc_fence_after();
    const float inv = some && l != 0.f ? 1.f / l : 0.f;             // no key: zero (NaN sums stay NaN)
    T* o_row = out + ((long long)row * g.Hq + h) * g.D;
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
          uint32_t w[8];
#pragma unroll
          for (int i = 0; i < 8; ++i)
            w[i] = Elem<T>::pack(inv == 0.f ? 0.f : __uint_as_float(o[16 * u + 2 * i]) * inv,
                                 inv == 0.f ? 0.f : __uint_as_float(o[16 * u + 2 * i + 1]) * inv);
          const int d0 = 32 * c + 16 * u;
          if (d0 + 16 <= g.D && (g.D & 15) == 0) {
            st_global_32(o_row + d0, w);
          } else if (d0 < g.D) {                                    // dims are a multiple of 8
            *reinterpret_cast<uint4*>(o_row + d0) = make_uint4(w[0], w[1], w[2], w[3]);
            if (d0 + 8 < g.D) *reinterpret_cast<uint4*>(o_row + d0 + 8) = make_uint4(w[4], w[5], w[6], w[7]);
          }
        }
      }
    }
    if (lse && row < g.T)
      lse[(long long)h * g.T + row] = inv == 0.f ? -INFINITY : (m + log2f(l)) * (1.f / LOG2E);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 8) tmem_dealloc(tm, 512);
  if (threadIdx.x == 0 && *serr) atomicExch(gerr, 1);
}

template <typename T, int DH>
int launch(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, void* o, float* lse, const Geo& g, int* err,
           cudaStream_t st) {
  auto kern = packed_fwd_kernel<T, DH>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<DH>::total);
  if (e != cudaSuccess) return (int)e;
  kern<<<dim3((unsigned)((long long)g.Hq * g.pairs)), NT, Cfg<DH>::total, st>>>(mq, mk, mv, (T*)o, lse, g, err);
  DMB_CHECK_LAUNCH();
  return 0;
}

}  // namespace

// q [T, Hq, D] (row stride, head stride), k / v [T, Hkv, D] likewise, 16-bit elements (half: fp16, else bf16); o [T, Hq, D]
// contiguous; lse [Hq, T] fp32 or null.  Strides are multiples of 8 elements, pointers 16-byte aligned, D a multiple of 8
// up to 128 (the caller checks).
extern "C" int dmb_packed_attn_fwd(const void* q, long long q_rs, long long q_hs, const void* k, long long k_rs, long long k_hs,
                                   const void* v, long long v_rs, long long v_hs, const int* cu, int nseq, void* o, float* lse,
                                   int T, int Hq, int Hkv, int D, int window, float scale, int half, int* err, void* stream) {
  if (T <= 0) return 0;
  if (D <= 0 || D > 128 || (D & 7) || Hkv <= 0 || Hq % Hkv || nseq < 0) return -1;
  CUtensorMap mq, mk, mv;
  int rc = bind_context();
  if (rc == 0) rc = make_map_rows(&mq, q, D, Hq, T, q_rs, q_hs);
  if (rc == 0) rc = make_map_rows(&mk, k, D, Hkv, T, k_rs, k_hs);
  if (rc == 0) rc = make_map_rows(&mv, v, D, Hkv, T, v_rs, v_hs);
  if (rc) return rc;
  const int pairs = (int)(((long long)T + 2 * TILE - 1) / (2 * TILE));
  if ((long long)pairs * Hq > 0x7fffffffLL) return -1;
  const Geo g{cu, nseq, T, Hq, Hq / Hkv, D, window, pairs, scale * LOG2E};
  cudaStream_t st = (cudaStream_t)stream;
  if (half) return D <= 64 ? launch<__half, 64>(mq, mk, mv, o, lse, g, err, st) : launch<__half, 128>(mq, mk, mv, o, lse, g, err, st);
  return D <= 64 ? launch<bf16, 64>(mq, mk, mv, o, lse, g, err, st) : launch<bf16, 128>(mq, mk, mv, o, lse, g, err, st);
}
