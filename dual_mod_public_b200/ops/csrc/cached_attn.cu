// Attention of one new token per sequence over a cache [B, P, Hkv, D] with a live length per sequence.
//
//   o_h = sum_{j in [lo, len)} softmax(scale q_h . k_j) v_j,   lo = max(0, len - window),   query heads h share key head h / g
//
// Bound by reading the live rows of K and V once.  A block takes a chunk of CHUNK keys of one (sequence, key head); its warps
// take tiles of 16 keys in turn, each warp with a ring of its own filled by asynchronous copies (no barrier between warps
// until the end).  All query heads of the group are the 16 rows of a warp-level MMA (m16n8k16): one head or sixteen, the keys
// are read once and the matrix pipe stays far below its rate, so padding the rows costs nothing that bounds.  Rows behind the
// live length are never read: they are filled with zeros in shared memory, whatever the cache holds there.
// Chunks of a sequence are joined by a second kernel in chunk order (no atomics); a call whose cache fits one chunk writes its
// output directly.
#include "packed.cuh"

namespace {

constexpr int WARPS = 4, KEYS = 16, STAGES = 4, ROWS = 16;

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
  int B, P, Hq, Hkv, group, D, window, chunk, splits;
  float scale_log2;
};

// live rows [lo, len) of a sequence
__device__ __forceinline__ int2 live_rows(const int* __restrict__ lengths, const Geo& g, int b) {
  const int len = min(g.P, max(0, __ldg(lengths + b)));
  return make_int2(g.window > 0 ? max(0, len - g.window) : 0, len);
}

template <int DH>
constexpr int smem_bytes() { return WARPS * STAGES * 2 * KEYS * DH * 2; }

template <typename T, int DH>
__global__ void __launch_bounds__(WARPS * 32) cached_kernel(const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v,
                                                            const int* __restrict__ lengths, T* __restrict__ out,
                                                            float* __restrict__ po, float2* __restrict__ pml, const Geo g) {
  using E = packed::Elem<T>;
  constexpr int RB = DH * 2;                              // bytes of a row in shared memory (16-byte chunks xor-swizzled)
  constexpr int CH = DH / 8;                              // 16-byte chunks per row
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rtiles = (g.group + ROWS - 1) / ROWS;
  const int split = blockIdx.x, kh = blockIdx.y / rtiles, rt = blockIdx.y % rtiles, b = blockIdx.z;
  const int2 lr = live_rows(lengths, g, b);
  const int k_begin = lr.x + split * g.chunk, k_end = min(lr.y, k_begin + g.chunk);
  const int heads = min(ROWS, g.group - rt * ROWS), h0 = kh * g.group + rt * ROWS;
  if (k_begin >= k_end && (g.splits > 1 || lr.y > lr.x)) return;         // the joining kernel does not look here
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
  const uint32_t ring = smem_u32(smem) + warp * (STAGES * 2 * KEYS * RB);
  const T* kp = k + b * g.k_bs + (long long)kh * g.k_hs;
  const T* vp = v + b * g.v_bs + (long long)kh * g.v_hs;
  const int tiles = k_end > k_begin ? (k_end - k_begin + KEYS - 1) / KEYS : 0;
  auto swz = [](int row, int c) { return row * RB + ((c ^ (row & 7)) << 4); };
  auto load = [&](int tile, int stage) {                   // this warp's tile-th tile
    if (tile < tiles) {
      const uint32_t dk = ring + stage * (2 * KEYS * RB), dv = dk + KEYS * RB;
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
    const uint32_t sk = ring + stage * (2 * KEYS * RB), sv = sk + KEYS * RB;
    float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f};    // keys 0..7 and 8..15 of the tile
#pragma unroll
    for (int s = 0; s < DH / 16; ++s) {
      uint32_t b0, b1, b2, b3;      // (keys 0..7, dims lo), (keys 0..7, dims hi), (keys 8..15, lo), (keys 8..15, hi)
      ldsm_x4(b0, b1, b2, b3, sk + swz((lane & 7) + ((lane >> 4) << 3), 2 * s + ((lane >> 3) & 1)));
      mma<T>(s0, qa[s], b0, b1);
      mma<T>(s1, qa[s], b2, b3);
    }
    const int left = k_end - (k_begin + t * KEYS);                       // live keys from the tile's first on
    uint32_t pa[4];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float x[4] = {s0[2 * r], s0[2 * r + 1], s1[2 * r], s1[2 * r + 1]};
      const int c0 = (lane & 3) * 2;
      if (left < KEYS) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (c0 + (i & 1) + (i >> 1) * 8 >= left) x[i] = -INFINITY;
      }
      const float top = quad_max(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]))) * g.scale_log2;
      const float mn = fmaxf(m[r], top), sub = mn == -INFINITY ? 0.f : mn;
      const float f = exp2f(m[r] - sub);
      m[r] = mn;
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = exp2f(fmaf(x[i], g.scale_log2, -sub));
      l[r] = l[r] * f + ((x[0] + x[1]) + (x[2] + x[3]));
      if (__any_sync(0xffffffffu, f != 1.f)) {
#pragma unroll
        for (int i = 0; i < DH / 8; ++i) {
          o[i][2 * r] *= f;
          o[i][2 * r + 1] *= f;
        }
      }
      pa[r] = E::pack(x[0], x[1]);
      pa[2 + r] = E::pack(x[2], x[3]);
    }
#pragma unroll
    for (int n = 0; n < DH / 16; ++n) {                                   // 16 dims per step
      uint32_t b0, b1, b2, b3;      // (keys 0..7, dims lo), (keys 8..15, lo), (keys 0..7, hi), (keys 8..15, hi), transposed
      ldsm_x4_t(b0, b1, b2, b3, sv + swz((lane & 7) + (((lane >> 3) & 1) << 3), 2 * n + (lane >> 4)));
      mma<T>(o[2 * n], pa, b0, b1);
      mma<T>(o[2 * n + 1], pa, b2, b3);
    }
    __syncwarp();
    stage = (stage + 1) % STAGES;
  }
  cp_async_wait<0>();
  __syncthreads();                                                        // the rings are free
  // ---- join the warps ----
  float* so = reinterpret_cast<float*>(smem);                            // [WARPS][ROWS][DH]
  __shared__ float sm[WARPS][ROWS], sl[WARPS][ROWS];
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
    for (int r = 0; r < 2; ++r) {
      float* d = so + (warp * ROWS + rA + 8 * r) * DH + 8 * i + (lane & 3) * 2;
      d[0] = o[i][2 * r];
      d[1] = o[i][2 * r + 1];
    }
  __syncthreads();
  for (int i = threadIdx.x; i < heads * (DH / 2); i += WARPS * 32) {
    const int r = i / (DH / 2), d = (i % (DH / 2)) * 2;
    float top = sm[0][r];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) top = fmaxf(top, sm[w][r]);
    const float sub = top == -INFINITY ? 0.f : top;
    float sum = 0.f, a0 = 0.f, a1 = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float f = exp2f(sm[w][r] - sub);
      sum = fmaf(f, sl[w][r], sum);
      a0 = fmaf(f, so[(w * ROWS + r) * DH + d], a0);
      a1 = fmaf(f, so[(w * ROWS + r) * DH + d + 1], a1);
    }
    if (d >= g.D) continue;
    const long long hrow = (long long)b * g.Hq + h0 + r;
    if (g.splits == 1) {
      const float inv = sum != 0.f ? 1.f / sum : 0.f;                     // no live row: zero
      *reinterpret_cast<uint32_t*>(out + hrow * g.D + d) = E::pack(inv == 0.f ? 0.f : a0 * inv, inv == 0.f ? 0.f : a1 * inv);
    } else {
      float* p = po + (hrow * g.splits + split) * g.D + d;
      *reinterpret_cast<float2*>(p) = make_float2(a0, a1);
      if (d == 0) pml[hrow * g.splits + split] = make_float2(top, sum);
    }
  }
}

// joins the chunks of one (sequence, query head): a warp per head, chunk order
template <typename T>
__global__ void __launch_bounds__(128) cached_join_kernel(const float* __restrict__ po, const float2* __restrict__ pml,
                                                          const int* __restrict__ lengths, T* __restrict__ out, const Geo g) {
  const long long hrow = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (hrow >= (long long)g.B * g.Hq) return;
  const int2 lr = live_rows(lengths, g, (int)(hrow / g.Hq));
  const int n = (lr.y - lr.x + g.chunk - 1) / g.chunk;
  float top = -INFINITY;
  for (int s = lane; s < n; s += 32) top = fmaxf(top, pml[hrow * g.splits + s].x);
  top = warp_max(top);
  const float sub = top == -INFINITY ? 0.f : top;
  float sum = 0.f, a[4] = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < n; ++s) {
    const float2 ml = pml[hrow * g.splits + s];
    const float f = exp2f(ml.x - sub);
    sum = fmaf(f, ml.y, sum);
    const float* p = po + (hrow * g.splits + s) * g.D;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int d = 64 * i + 2 * lane;
      if (d < g.D) {
        const float2 w = *reinterpret_cast<const float2*>(p + d);
        a[2 * i] = fmaf(f, w.x, a[2 * i]);
        a[2 * i + 1] = fmaf(f, w.y, a[2 * i + 1]);
      }
    }
  }
  const float inv = sum != 0.f ? 1.f / sum : 0.f;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int d = 64 * i + 2 * lane;
    if (d < g.D)
      *reinterpret_cast<uint32_t*>(out + hrow * g.D + d) =
          packed::Elem<T>::pack(inv == 0.f ? 0.f : a[2 * i] * inv, inv == 0.f ? 0.f : a[2 * i + 1] * inv);
  }
}

template <typename T, int DH>
int launch(const void* q, const void* k, const void* v, const int* lengths, void* o, float* po, float2* pml, const Geo& g,
           cudaStream_t st) {
  auto kern = cached_kernel<T, DH>;
  constexpr int smem = smem_bytes<DH>();
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return (int)e;
  const int rtiles = (g.group + ROWS - 1) / ROWS;
  kern<<<dim3(g.splits, g.Hkv * rtiles, g.B), WARPS * 32, smem, st>>>((const T*)q, (const T*)k, (const T*)v, lengths, (T*)o, po, pml, g);
  DMB_CHECK_LAUNCH();
  if (g.splits > 1) {
    const long long rows = (long long)g.B * g.Hq;
    cached_join_kernel<T><<<(unsigned)((rows + 3) / 4), 128, 0, st>>>(po, pml, lengths, (T*)o, g);
    DMB_CHECK_LAUNCH();
  }
  return 0;
}

}  // namespace

// q [B, Hq, D], k / v [B, P, Hkv, D] by strides (elements; multiples of 8 except that q's may be any even), 16-bit elements
// (half: fp16, else bf16); o [B, Hq, D] contiguous.  chunk: keys per block, splits = chunks that cover the longest live range;
// po fp32 [B, Hq, splits, D] and pml fp32 [B, Hq, splits, 2] when splits > 1, else unused.
extern "C" int dmb_cached_attn(const void* q, long long q_bs, long long q_hs, const void* k, long long k_bs, long long k_rs,
                               long long k_hs, const void* v, long long v_bs, long long v_rs, long long v_hs, const int* lengths,
                               void* o, float* po, float* pml, int B, int P, int Hq, int Hkv, int D, int window, int chunk,
                               int splits, float scale, int half, void* stream) {
  if (B <= 0) return 0;
  if (P < 0 || D <= 0 || D > 128 || (D & 7) || Hkv <= 0 || Hq % Hkv || splits < 1 || chunk < KEYS || B > 65535) return -1;
  const Geo g{q_bs, q_hs, k_bs, k_rs, k_hs, v_bs, v_rs, v_hs, B, P, Hq, Hkv, Hq / Hkv, D, window, chunk, splits,
              scale * packed::LOG2E};
  if ((long long)Hkv * ((g.group + ROWS - 1) / ROWS) > 65535) return -1;
  cudaStream_t st = (cudaStream_t)stream;
  float2* ml = (float2*)pml;
  if (half)
    return D <= 64 ? launch<__half, 64>(q, k, v, lengths, o, po, ml, g, st) : launch<__half, 128>(q, k, v, lengths, o, po, ml, g, st);
  return D <= 64 ? launch<bf16, 64>(q, k, v, lengths, o, po, ml, g, st) : launch<bf16, 128>(q, k, v, lengths, o, po, ml, g, st);
}
