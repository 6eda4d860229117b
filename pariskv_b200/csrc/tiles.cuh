// What the tiled attention kernels for several tokens a step share.
#pragma once
#include "attend.cuh"
#include "tma.cuh"

namespace pk {

__device__ __forceinline__ float ex2(float x) {   // 2^x, results below 2^-126 are zero
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// (a + c) f, (b + c) f: two fp32 operations in one instruction
__device__ __forceinline__ void add_mul2(float& a, float& b, float c, float f) {
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 y, {%2, %2};\n\tadd.rn.f32x2 x, x, y;\n\tmov.b64 y, {%3, %3};\n\tmul.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "+f"(a), "+f"(b)
      : "f"(c), "f"(f));
}
__device__ __forceinline__ void add2(float& a, float& b, float c, float d) {
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 y, {%2, %3};\n\tadd.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "+f"(a), "+f"(b)
      : "f"(c), "f"(d));
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ void wait_ld(uint32_t (&r)[32]) {   // the values are there behind it, and no use of them moves before it
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                 "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                 "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])::"memory");
}
__device__ __forceinline__ void named_barrier(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
__device__ __forceinline__ bool not_finite(uint32_t bf16) { return (bf16 & 0x7f80u) == 0x7f80u; }

// ---- equal ranges of the tiles of all items, laid end to end; the lengths come from device memory ----
// Where the range of block i of `shares` begins, and which block has tile x.
__device__ __forceinline__ int64_t share_begin(int64_t total, unsigned i, unsigned shares) {
  return total < 1 << 22 ? (unsigned)total * i / shares : total * i / shares;   // (a division of 64 bits takes a hundred clocks)
}
__device__ __forceinline__ int share_owner(int64_t x, int64_t total, unsigned shares) {
  return total < 1 << 22 ? (int)(((unsigned)(x + 1) * shares - 1) / (unsigned)total) : (int)(((x + 1) * shares - 1) / total);
}
// Joins n partial results of a query row, record(i) = O rows of 128, then `rows` values m (log2), then `rows` sums l, in the order of i: a block of 128
// threads.  A warp takes every fourth record, four channels a lane, eight loads in flight; latency is what bounds it.  ALL: a record whose weight is zero counts too, so that what is not a number in it
// is not lost; every record then has to have been written.
struct MergeShared {
  float o[4][128], l[4];
};
template <bool ALL = false, class Record>
__device__ __forceinline__ void merge_row(MergeShared& s, int n, int rows, int r, Record record, uint16_t* out, float* lse) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  float M = -INFINITY;
  for (int i = lane; i < n; i += 32) M = fmaxf(M, record(i)[rows * 128 + r]);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, off));
  float L = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  const int mine = (n - warp + 3) / 4;   // records of this warp
  for (int i0 = 0; i0 < mine; i0 += 32) {
    float f = 0.0f;
    if (i0 + lane < mine) {
      const float* rec = record(4 * (i0 + lane) + warp);
      const float m = rec[rows * 128 + r];
      f = m == -INFINITY ? 0.0f : exp2f(m - M);
      L += rec[rows * 129 + r] * f;
    }
    const int cnt = min(32, mine - i0);
    for (int k0 = 0; k0 < cnt; k0 += 8) {
      float4 v[8];
#pragma unroll
      for (int k = 0; k < 8; k++)
        v[k] = k0 + k < cnt ? *reinterpret_cast<const float4*>(record(4 * (i0 + k0 + k) + warp) + (int64_t)r * 128 + 4 * lane) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int k = 0; k < 8; k++) {
        const float fk = __shfl_sync(0xffffffffu, f, k0 + k);
        if (k0 + k < cnt && (ALL || fk != 0.0f)) o[0] += v[k].x * fk, o[1] += v[k].y * fk, o[2] += v[k].z * fk, o[3] += v[k].w * fk;   // (NaN != 0)
      }
    }
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) L += __shfl_xor_sync(0xffffffffu, L, off);
  *reinterpret_cast<float4*>(&s.o[warp][4 * lane]) = make_float4(o[0], o[1], o[2], o[3]);
  if (lane == 0) s.l[warp] = L;
  __syncthreads();
  L = (s.l[0] + s.l[1]) + (s.l[2] + s.l[3]);
  const float O = (s.o[0][tid] + s.o[1][tid]) + (s.o[2][tid] + s.o[3][tid]);
  out[tid] = f2bf(L == 0.0f ? 0.0f : O / L);
  if (lse && tid == 0) *lse = L == 0.0f ? -INFINITY : M + log2f(L);
}

// Rows of 128 bf16 in three dimensions, boxes of 64 channels x `box` rows; false where a tensor map cannot have these strides.
inline bool rows_map(CUtensorMap* m, const void* base, int64_t d1, int64_t s1, int64_t d2, int64_t s2, int64_t d3, int64_t s3, int box) {
  const auto encode = tensor_map_encoder();
  const int64_t d[3] = {d1, d2, d3};
  int64_t s[3] = {s1, s2, s3};
  for (int i = 0; i < 3; i++) {
    if (d[i] == 1) s[i] = 128;
    if (s[i] <= 0 || s[i] >= (1ll << 38) || d[i] >= (1ll << 31)) return false;
  }
  if (!encode) return false;
  const cuuint64_t dims[4] = {128, (cuuint64_t)d1, (cuuint64_t)d2, (cuuint64_t)d3}, strides[3] = {(cuuint64_t)s[0] * 2, (cuuint64_t)s[1] * 2, (cuuint64_t)s[2] * 2};
  const cuuint32_t boxes[4] = {64, (cuuint32_t)box, 1, 1}, steps[4] = {1, 1, 1, 1};
  return encode(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides, boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}


}  // namespace pk
