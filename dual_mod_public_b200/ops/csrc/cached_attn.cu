// Attention of one new token per sequence over a cache [B, P, Hkv, D] with a live length per sequence.
//
//   o_h = sum_{j in [lo, len)} softmax(scale q_h . k_j) v_j,   lo = max(0, len - window),   query heads h share key head h / g
//
// Bound by reading the live rows of K and V once (64 sequences of up to 8192 rows, 16 query and 4 key heads of 128: 90 us, 5.6
// TB/s; one sequence of 1190 rows, 16 heads of 64: 8.4 us, all of it latency).  A cluster of 1 to 16 blocks shares the live rows of one (sequence, key head)
// out evenly; a block's warps take tiles of KEYS keys in turn, each warp with a ring of its own filled by asynchronous copies
// (no barrier between warps until the end).  All query heads of the group are the 16 rows of a warp-level MMA (m16n8k16): one
// head or sixteen, the keys are read once and the matrix pipe stays far below its rate, so padding the rows costs nothing that
// bounds.  Rows behind the live length are never read: they are filled with zeros in shared memory, whatever the cache holds
// there.  The blocks of a cluster join their parts through each other's shared memory, in block order: one launch, no
// workspace, no atomics.
#include <climits>

#include "packed.cuh"

namespace {

constexpr int WARPS = 4, STAGES = 2, ROWS = 16, MAX_CLUSTER = 16;

template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma<bf16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  mma16816(d, a, b0, b1);
}
template <>
__device__ __forceinline__ void mma<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// 16 bytes, or zeros where `live` is false (nothing is read then)
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}

struct Geo {
  long long q_bs, q_hs, k_bs, k_rs, k_hs, v_bs, v_rs, v_hs;
  int P, Hq, group, D, window;
  float scale_log2;
};

template <int DH>
struct Cfg {
  static constexpr int KEYS = DH == 64 ? 32 : 16;          // keys of a tile: 8 KB of K and V
  static constexpr int RB = DH * 2, CH = DH / 8;           // bytes and 16-byte chunks of a row in shared memory
  static constexpr int TILE_B = KEYS * RB, smem = WARPS * STAGES * 2 * TILE_B;
};

__device__ __forceinline__ float ld_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float2 ld_cluster2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}

template <typename T, int DH>
__global__ void __launch_bounds__(WARPS * 32) cached_kernel(const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v,
                                                            const int* __restrict__ lengths, T* __restrict__ out, const Geo g) {
  using E = packed::Elem<T>;
  using C = Cfg<DH>;
  constexpr int KEYS = C::KEYS, RB = C::RB, CH = C::CH;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rtiles = (g.group + ROWS - 1) / ROWS, blocks = gridDim.x;               // the cluster is the grid's first axis
  const int part = blockIdx.x, kh = blockIdx.y / rtiles, rt = blockIdx.y % rtiles, b = blockIdx.z;
  const int heads = min(ROWS, g.group - rt * ROWS), h0 = kh * g.group + rt * ROWS;
  const int len = min(g.P, max(0, __ldg(lengths + b)));
  // ---- the group's queries as the A operand ----
  uint32_t qa[DH / 16][4];
  {
    const int r0 = lane >> 2, c0 = (lane & 3) * 2;
#pragma unroll
    for (int s = 0; s < DH / 16; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = r0 + (i & 1) * 8, d = 16 * s + c0 + (i >> 1) * 8;
        qa[s][i] = r < heads && d < g.D
                       ? *reinterpret_cast<const uint32_t*>(q + b * g.q_bs + (long long)(h0 + r) * g.q_hs + d) : 0u;
      }
  }
  // this block's share of the live rows [len - window, len), in whole tiles per warp
  const int first = g.window > 0 ? max(0, len - g.window) : 0;
  const int share = ((len - first + blocks - 1) / blocks + KEYS - 1) / KEYS * KEYS;
  const int k_begin = min(len, first + part * share), k_end = min(len, k_begin + share);
  const uint32_t ring = smem_u32(smem) + warp * (STAGES * 2 * C::TILE_B);
  const T* kp = k + b * g.k_bs + (long long)kh * g.k_hs;
  const T* vp = v + b * g.v_bs + (long long)kh * g.v_hs;
  const int tiles = (k_end - k_begin + KEYS - 1) / KEYS;
  auto swz = [](int row, int c) { return row * RB + ((c ^ (row & 7)) << 4); };
  auto load = [&](int tile, int stage) {
    if (tile < tiles) {
      const uint32_t dk = ring + stage * (2 * C::TILE_B), dv = dk + C::TILE_B;
      const int r0 = k_begin + tile * KEYS;
#pragma unroll
      for (int i = lane; i < KEYS * CH; i += 32) {
        const int r = i / CH, c = i % CH;
        const bool live = r0 + r < k_end && c * 8 < g.D;
        const long long row = live ? r0 + r : 0;
        const int d = live ? c * 8 : 0;
        copy16(dk + swz(r, c), kp + row * g.k_rs + d, live);
        copy16(dv + swz(r, c), vp + row * g.v_rs + d, live);
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) load(warp + s * WARPS, s);
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, o[DH / 8][4];
#pragma unroll
  for (int i = 0; i < DH / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  int stage = 0;
  for (int t = warp; t < tiles; t += WARPS) {
    load(t + (STAGES - 1) * WARPS, (stage + STAGES - 1) % STAGES);
    cp_async_wait<STAGES - 1>();
    __syncwarp();
    const uint32_t sk = ring + stage * (2 * C::TILE_B), sv = sk + C::TILE_B;
    float x[KEYS / 8][4];                                                // scores: 8 keys each
#pragma unroll
    for (int n = 0; n < KEYS / 8; ++n) x[n][0] = x[n][1] = x[n][2] = x[n][3] = 0.f;
#pragma unroll
    for (int s = 0; s < DH / 16; ++s)
#pragma unroll
      for (int n = 0; n < KEYS / 16; ++n) {
        uint32_t b0, b1, b2, b3;    // (keys 0..7, dims lo), (keys 0..7, dims hi), (keys 8..15, lo), (keys 8..15, hi)
        ldsm_x4(b0, b1, b2, b3, sk + swz(16 * n + (lane & 7) + ((lane >> 4) << 3), 2 * s + ((lane >> 3) & 1)));
        mma<T>(x[2 * n], qa[s], b0, b1);
        mma<T>(x[2 * n + 1], qa[s], b2, b3);
      }
    const int left = k_end - (k_begin + t * KEYS);                       // live keys from the tile's first on
    uint32_t pa[KEYS / 16][4];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float top = -INFINITY;
#pragma unroll
      for (int n = 0; n < KEYS / 8; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (left < KEYS && 8 * n + (lane & 3) * 2 + i >= left) x[n][2 * r + i] = -INFINITY;
          top = fmaxf(top, x[n][2 * r + i]);
        }
      // m is a score, and differences of scores are formed before the factor: exact next to the maximum however large it is
      const float mn = fmaxf(m[r], quad_max(top)), sub = mn == -INFINITY ? 0.f : mn;
      const float f = exp2f((m[r] - sub) * g.scale_log2);
      m[r] = mn;
      float sum = 0.f;
#pragma unroll
      for (int n = 0; n < KEYS / 8; ++n) {
        const float p0 = exp2f((x[n][2 * r] - sub) * g.scale_log2), p1 = exp2f((x[n][2 * r + 1] - sub) * g.scale_log2);
        sum += p0 + p1;
        pa[n >> 1][r + 2 * (n & 1)] = E::pack(p0, p1);
      }
      l[r] = l[r] * f + sum;
      if (__any_sync(0xffffffffu, f != 1.f)) {
#pragma unroll
        for (int i = 0; i < DH / 8; ++i) {
          o[i][2 * r] *= f;
          o[i][2 * r + 1] *= f;
        }
      }
    }
#pragma unroll
    for (int d = 0; d < DH / 16; ++d)                                     // 16 dims per step
#pragma unroll
      for (int n = 0; n < KEYS / 16; ++n) {
        uint32_t b0, b1, b2, b3;    // (keys 0..7, dims lo), (keys 8..15, lo), (keys 0..7, hi), (keys 8..15, hi), transposed
        ldsm_x4_t(b0, b1, b2, b3, sv + swz(16 * n + (lane & 7) + (((lane >> 3) & 1) << 3), 2 * d + (lane >> 4)));
        mma<T>(o[2 * d], pa[n], b0, b1);
        mma<T>(o[2 * d + 1], pa[n], b2, b3);
      }
    __syncwarp();
    stage = (stage + 1) % STAGES;
  }
  cp_async_wait<0>();
  __syncthreads();                                                        // the rings are free
  // ---- join the warps ----
  float* so = reinterpret_cast<float*>(smem);                            // [WARPS][ROWS][DH], then the block's [ROWS][DH] in front
  __shared__ float sm[WARPS][ROWS], sl[WARPS][ROWS], bm[ROWS], bl[ROWS];
  l[0] = quad_sum(l[0]);
  l[1] = quad_sum(l[1]);
  const int rA = lane >> 2;
  if ((lane & 3) == 0) {
    sm[warp][rA] = m[0]; sm[warp][rA + 8] = m[1];
    sl[warp][rA] = l[0]; sl[warp][rA + 8] = l[1];
  }
#pragma unroll
  for (int i = 0; i < DH / 8; ++i)
#pragma unroll
    for (int r = 0; r < 2; ++r)
      if (rA + 8 * r < heads)
        *reinterpret_cast<float2*>(so + (warp * ROWS + rA + 8 * r) * DH + 8 * i + (lane & 3) * 2) =
            make_float2(o[i][2 * r], o[i][2 * r + 1]);
  __syncthreads();
  for (int i = threadIdx.x; i < heads * (DH / 2); i += WARPS * 32) {
    const int r = i / (DH / 2), d = (i % (DH / 2)) * 2;
    float top = sm[0][r];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) top = fmaxf(top, sm[w][r]);
    const float sub = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
    float2 a = make_float2(0.f, 0.f);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float f = exp2f((sm[w][r] - sub) * g.scale_log2);
      const float2 u = *reinterpret_cast<const float2*>(so + (w * ROWS + r) * DH + d);
      sum = fmaf(f, sl[w][r], sum);
      a.x = fmaf(f, u.x, a.x);
      a.y = fmaf(f, u.y, a.y);
    }
    if (blocks == 1) {
      const float inv = sum != 0.f ? 1.f / sum : 0.f;                     // no live row: zero
      if (d < g.D)
        *reinterpret_cast<uint32_t*>(out + ((long long)b * g.Hq + h0 + r) * g.D + d) =
            E::pack(inv == 0.f ? 0.f : a.x * inv, inv == 0.f ? 0.f : a.y * inv);
    } else {
      *reinterpret_cast<float2*>(so + r * DH + d) = a;                    // this thread alone reads and writes these
      if (d == 0) { bm[r] = top; bl[r] = sum; }
    }
  }
  if (blocks == 1) return;
  // ---- join the blocks: each takes a slice of the outputs ----
  tc05::cluster_sync_all();
  const uint32_t so_a = smem_u32(so), bm_a = smem_u32(bm), bl_a = smem_u32(bl);
  for (int i = part * (WARPS * 32) + threadIdx.x; i < heads * (DH / 2); i += blocks * (WARPS * 32)) {
    const int r = i / (DH / 2), d = (i % (DH / 2)) * 2;
    float mb[MAX_CLUSTER], top = -INFINITY;
#pragma unroll
    for (int w = 0; w < MAX_CLUSTER; ++w) {
      mb[w] = w < blocks ? ld_cluster(tc05::map_to_cta(bm_a + 4 * r, w)) : -INFINITY;
      top = fmaxf(top, mb[w]);
    }
    const float sub = top == -INFINITY ? 0.f : top;
    float sum = 0.f, a0 = 0.f, a1 = 0.f;
#pragma unroll
    for (int w = 0; w < MAX_CLUSTER; ++w)
      if (w < blocks) {
        const float f = exp2f((mb[w] - sub) * g.scale_log2);
        const float2 u = ld_cluster2(tc05::map_to_cta(so_a + 4 * (r * DH + d), w));
        sum = fmaf(f, ld_cluster(tc05::map_to_cta(bl_a + 4 * r, w)), sum);
        a0 = fmaf(f, u.x, a0);
        a1 = fmaf(f, u.y, a1);
      }
    const float inv = sum != 0.f ? 1.f / sum : 0.f;
    if (d < g.D)
      *reinterpret_cast<uint32_t*>(out + ((long long)b * g.Hq + h0 + r) * g.D + d) =
          E::pack(inv == 0.f ? 0.f : a0 * inv, inv == 0.f ? 0.f : a1 * inv);
  }
  tc05::cluster_sync_all();                                               // nobody leaves while its memory is read
}

template <typename T, int DH>
int launch(const void* q, const void* k, const void* v, const int* lengths, void* o, int B, int Hkv, int blocks, const Geo& g,
           cudaStream_t st) {
  auto kern = cached_kernel<T, DH>;
  static std::atomic<unsigned long long> set{0};
  if (int rc = packed::allow_smem(kern, Cfg<DH>::smem, set)) return rc;
  cudaError_t e = cudaSuccess;
  if (blocks > 8) e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e != cudaSuccess) return (int)e;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = blocks;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks, Hkv * ((g.group + ROWS - 1) / ROWS), B);
  cfg.blockDim = dim3(WARPS * 32);
  cfg.dynamicSmemBytes = Cfg<DH>::smem;
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = blocks > 1 ? 1 : 0;
  e = cudaLaunchKernelEx(&cfg, kern, (const T*)q, (const T*)k, (const T*)v, lengths, (T*)o, g);
  if (e != cudaSuccess) return (int)e;
  DMB_CHECK_LAUNCH();
  return 0;
}

}  // namespace

// q [B, Hq, D], k / v [B, P, Hkv, D] by strides (elements; multiples of 8 except that q's may be any even), 16-bit elements
// (half: fp16, else bf16); o [B, Hq, D] contiguous; blocks: 1, 2, 4, 8 or 16 that share a sequence's rows of one key head.
extern "C" int dmb_cached_attn(const void* q, long long q_bs, long long q_hs, const void* k, long long k_bs, long long k_rs,
                               long long k_hs, const void* v, long long v_bs, long long v_rs, long long v_hs, const int* lengths,
                               void* o, int B, int P, int Hq, int Hkv, int D, int window, int blocks, float scale, int half,
                               void* stream) {
  if (B <= 0) return 0;
  if (P < 0 || P > INT_MAX - 4095 || D <= 0 || D > 128 || (D & 7) || Hkv <= 0 || Hq % Hkv || B > 65535) return -1;
  if (blocks < 1 || blocks > MAX_CLUSTER || (blocks & (blocks - 1))) return -1;
  const Geo g{q_bs, q_hs, k_bs, k_rs, k_hs, v_bs, v_rs, v_hs, P, Hq, Hq / Hkv, D, window, scale * packed::LOG2E};
  if ((long long)Hkv * ((g.group + ROWS - 1) / ROWS) > 65535) return -1;
  cudaStream_t st = (cudaStream_t)stream;
  if (half)
    return D <= 64 ? launch<__half, 64>(q, k, v, lengths, o, B, Hkv, blocks, g, st) : launch<__half, 128>(q, k, v, lengths, o, B, Hkv, blocks, g, st);
  return D <= 64 ? launch<bf16, 64>(q, k, v, lengths, o, B, Hkv, blocks, g, st) : launch<bf16, 128>(q, k, v, lengths, o, B, Hkv, blocks, g, st);
}
