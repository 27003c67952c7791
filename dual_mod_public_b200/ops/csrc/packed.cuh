// Helpers of the attention over packed sequences (packed_attn_fwd.cu, packed_attn_bwd.cu): which keys a row of the packed
// axis sees, tile loads of [row, head, dim] tensors, and the tensor-memory operand forms of tcgen05.
#pragma once
#include <cuda_fp16.h>

#include <atomic>

#include "tc05.cuh"

namespace packed {

using namespace tc05;

constexpr int TILE = 128;               // rows of a query tile and of a key block
constexpr float LOG2E = 1.4426950408889634f;
constexpr float FAR = 16777216.f;       // octaves: fp32 holds a row's maximum or log sum to within one up to here

// ---- sequences -------------------------------------------------------------------------------------------------------
// `cu` holds n + 1 ascending row numbers; sequence s is the rows [cu[s], cu[s + 1]).  A row outside [cu[0], cu[n]) belongs
// to no sequence.  The values live on the device and are not checked there: every result is clamped, so a wrong table
// gives wrong outputs but no access out of range.

// first index whose entry is greater than `row` (0 .. n + 1)
__device__ __forceinline__ int upper_index(const int* __restrict__ cu, int n, int row) {
  int a = 0, b = n + 1;
  while (a < b) {
    const int m = (a + b) >> 1;
    if (__ldg(cu + m) > row) b = m; else a = m + 1;
  }
  return a;
}
// first key that query `row` sees (row + 1: none)
__device__ __forceinline__ int first_key(const int* __restrict__ cu, int n, int window, int row) {
  const int u = upper_index(cu, n, row);
  if (u == 0 || u == n + 1) return row + 1;
  int lo = min(row, max(0, __ldg(cu + u - 1)));
  if (window > 0) lo = max(lo, row - window + 1);
  return lo;
}
// last query that sees key `row` (row - 1: none)
__device__ __forceinline__ int last_query(const int* __restrict__ cu, int n, int window, int rows, int row) {
  const int u = upper_index(cu, n, row);
  if (u == 0 || u == n + 1) return row - 1;
  int hi = max(row, min(rows, __ldg(cu + u)) - 1);
  if (window > 0) hi = (int)min((long long)hi, (long long)row + window - 1);
  return hi;
}

// bits i of 32 columns c0 + i that lie in [lo, hi].  Masks are applied as tests of constant bits of such a word, which the
// hardware turns into predicates seven at a time: one select per element instead of two comparisons and a select (half of the
// blocks of documents of some hundred tokens hold a border; 8192 rows of eleven, 16 heads of 64, forward: 60 against 53 us).
__device__ __forceinline__ uint32_t range_bits(int c0, int lo, int hi) {
  const int a = max(lo - c0, 0), b = min(hi - c0, 31);
  return a > b ? 0u : (0xffffffffu >> (31 - b)) & (0xffffffffu << a);
}

// ---- waits and issue --------------------------------------------------------------------------------------------------
// A wait of a whole warp, bounded like mbar_wait: when it runs out it raises *err, and every later wait of the block returns
// at once, so the roles run to their ends on whatever lies in shared and tensor memory (all addresses stay in range) and the
// block reports the error.  One try comes before the clock is read: most waits of a running pipeline are over when asked for.
// No result and no vote: what follows stays warp-uniform for the compiler, which puts the operands of the tcgen05
// instructions into uniform registers only then (issuing one took 80 cycles otherwise).
__device__ __forceinline__ void wait(uint32_t bar, uint32_t parity, volatile int* err) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  if (!ok) mbar_wait(bar, parity, err);
  __syncwarp();
}
// true in one lane of a converged warp, always the same one
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r != 0;
}
// after a wait that ran out: an issuing warp lets its products in flight end before tensor memory is released
__device__ __forceinline__ void drain_products(uint32_t bar, volatile int* err) {
  if (!*err) return;
  volatile int ignore = 0;
  if (elect_one()) umma_commit(bar);
  __syncwarp();
  mbar_wait(bar, 0, &ignore);
}
// a value that is the same in all lanes, known as such to the compiler
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }

// ---- element types ----------------------------------------------------------------------------------------------------
template <typename T>
struct Elem;
template <>
struct Elem<bf16> {
  static constexpr uint32_t fmt = 1;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_bf16(lo, hi); }
  static __device__ __forceinline__ float2 unpack(uint32_t u) { return unpack_bf16(u); }
};
template <>
struct Elem<__half> {
  static constexpr uint32_t fmt = 0;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t u) {
    return __half22float2(*reinterpret_cast<__half2*>(&u));
  }
};
// instruction descriptor of kind::f16, both operands of type T, fp32 accumulator (instr_desc of tc05.cuh is bf16 only)
template <typename T>
__host__ __device__ constexpr uint32_t mma_desc(int m, int n, int a_mn, int b_mn) {
  return (1u << 4) | (Elem<T>::fmt << 7) | (Elem<T>::fmt << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// ---- tcgen05 ----------------------------------------------------------------------------------------------------------
// D (+)= A B with A in tensor memory: 128 lanes, two 16-bit elements per 32-bit column, 8 columns per K step of 16
__device__ __forceinline__ void umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t db, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(tmem_d), "r"(tmem_a), "l"(db), "r"(idesc), "r"(accumulate)
      : "memory");
}
// this thread's TMEM lane, 32 consecutive 32-bit columns starting at `taddr`
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]),
        "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]),
        "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
// the same with 16 columns
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// 16 lanes x 128 bits, 16 repetitions along the columns (32 registers): repetition j covers the 32-bit columns [4j, 4j + 4);
// thread t holds lane t/4, column 4j + t%4 in r[2j] and lane t/4 + 8 in r[2j + 1]: the pairs of 16-bit elements of the fragment
// that tmem_ld_16x256b_x16 (tc05.cuh) hands out
__device__ __forceinline__ void tmem_st_16x128b_x16(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x128b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// A tile of 128 rows x DH dims lies in shared memory as DH / 64 slabs of 128 rows x 128 bytes (128-byte swizzle).  The same
// tile serves as an operand whose reduction runs over the dims (K-major: 32 bytes per step of 16, 8-row groups 1024 bytes
// apart) and as one whose reduction runs over the rows (MN-major: 2048 bytes per step of 16 rows, slabs 16 KB apart).
constexpr uint32_t SLAB = TILE * 128;
__device__ __forceinline__ uint64_t desc_dims(uint32_t tile, int k) {
  return make_desc(tile + (k / 4) * SLAB + (k % 4) * 32, 16, 1024);
}
__device__ __forceinline__ uint64_t desc_rows(uint32_t tile, int k) { return make_desc(tile + k * 2048, SLAB, 1024); }
// what step k adds to the descriptor of step 0 (addresses count 16 bytes and stay below 2^18, so nothing carries over)
__device__ __forceinline__ constexpr uint64_t dims_step(int k) { return ((k / 4) * SLAB + (k % 4) * 32) >> 4; }
__device__ __forceinline__ constexpr uint64_t rows_step(int k) { return (k * 2048) >> 4; }

template <int DH>
__device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap* map, uint32_t bar, int head, int row) {
#pragma unroll
  for (int s = 0; s < DH / 64; ++s) tma_load_3d(dst + s * SLAB, map, bar, 64 * s, head, row);
}

// Zero the rows of a tile that belong to no sequence (their contents are the caller's padding and may be anything, and
// 0 x NaN would reach the product).  A whole warp; row0: the packed row of the tile's first row.
template <int DH>
__device__ __forceinline__ void blank_rows(uint8_t* tile, int row0, int begin, int end, int lane) {
  for (int r = 0; r < TILE; ++r) {
    if (row0 + r >= begin && row0 + r < end) continue;
    for (int c = lane; c < DH / 8; c += 32)
      *reinterpret_cast<uint4*>(tile + (c / 8) * SLAB + r * 128 + (c % 8) * 16) = make_uint4(0, 0, 0, 0);
  }
  fence_async_smem();
  __syncwarp();
}

// 32 bytes of one row per store: a full sector, although neighbouring threads write different rows
__device__ __forceinline__ void st_global_32(void* p, const uint32_t (&v)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]),
               "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

// ---- pairs of fp32 ----------------------------------------------------------------------------------------------------
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pair(float lo, float hi) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void split(f32x2 v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float ex2(float v) {               // special-function unit; results below 2^-126 are zero
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// 2^y of a pair on the FMA pipe, for y <= 126 (below -126, and for NaN: 2^-126).  y = n + f with n = round(y), |f| <= 1/2; 2^f by the
// minimax polynomial of degree 4 in relative error (Remez exchange on [-1/2, 1/2]: 2.7e-6), n added to the exponent field.
__device__ __forceinline__ void ex2_pair(f32x2 y, float& lo, float& hi) {
  float a, b;
  split(y, a, b);
  y = pair(fmaxf(a, -126.f), fmaxf(b, -126.f));
  const f32x2 magic = pair(12582912.f, 12582912.f);           // 1.5 x 2^23: its sum with y holds n in the low bits
  const f32x2 r = add2(y, magic);
  const f32x2 n = add2(r, pair(-12582912.f, -12582912.f));
  const f32x2 f = fma2(n, pair(-1.f, -1.f), y);
  f32x2 p = fma2(f, pair(0.009570102207362652f, 0.009570102207362652f), pair(0.05591785907745361f, 0.05591785907745361f));
  p = fma2(p, f, pair(0.240247443318367f, 0.240247443318367f));
  p = fma2(p, f, pair(0.6931217908859253f, 0.6931217908859253f));
  p = fma2(p, f, pair(0.9999992847442627f, 0.9999992847442627f));
  float pa, pb, ra, rb;
  split(p, pa, pb);
  split(r, ra, rb);
  lo = __uint_as_float(__float_as_uint(pa) + (__float_as_uint(ra) << 23));
  hi = __uint_as_float(__float_as_uint(pb) + (__float_as_uint(rb) << 23));
}
// maximum that is NaN when any operand is
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// ---- host -------------------------------------------------------------------------------------------------------------
// The driver call that encodes tensor maps wants a current context, and a thread that has made no runtime call yet (autograd
// runs backward passes on threads of its own) has none: naming the thread's device makes it current.
inline int bind_context() {
  int d = 0;
  cudaError_t e = cudaGetDevice(&d);
  if (e == cudaSuccess) e = cudaSetDevice(d);
  return (int)e;
}

// dynamic shared memory of a kernel, set once per device (`set`: a bit per device, one word per kernel)
template <typename K>
inline int allow_smem(K kernel, int bytes, std::atomic<unsigned long long>& set) {
  int d = 0;
  cudaError_t e = cudaGetDevice(&d);
  if (e != cudaSuccess) return (int)e;
  if (d < 64 && (set.load(std::memory_order_relaxed) >> d & 1)) return 0;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && d < 64) set.fetch_or(1ull << d, std::memory_order_relaxed);
  return (int)e;
}

// element (row, head, dim) of a 16-bit tensor at row * rs + head * hs + dim (strides in elements); boxes of 128 rows x 64
// dims of one head, dims and rows outside the tensor read as zero
inline int make_map_rows(CUtensorMap* m, const void* ptr, int dims, int heads, long long rows, long long rs, long long hs) {
  EncodeFn enc = encode_fn();
  if (!enc) return -10;
  cuuint64_t shape[3] = {(cuuint64_t)dims, (cuuint64_t)heads, (cuuint64_t)rows};
  cuuint64_t strides[2] = {(cuuint64_t)hs * 2, (cuuint64_t)rs * 2};
  cuuint32_t box[3] = {64, 1, TILE};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(ptr), shape, strides, box, estr,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : -11;
}

}  // namespace packed
