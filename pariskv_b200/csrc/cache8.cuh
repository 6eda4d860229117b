// The cache in 8 bits as its kernels see it: codes of whole blocks with a scale per block, and the last rows in 16 bits.
#pragma once
#include "attend.cuh"

namespace pk {

struct Cache8 {
  uint8_t* codes;
  int64_t c_b, c_h, c_l, c_kv;   // strides in codes
  float* scales;
  int64_t s_b, s_h, s_j, s_kv;
  uint16_t* recent;
  int64_t r_b, r_h, r_l, r_kv;
  int64_t cap;
  int R, shift, H;               // places of `recent`; log2 of the block
};

// Whether no two elements share memory: a dimension's step reaches behind all that the smaller steps span.
inline bool apart(const pk_tensor* t) {
  bool used[PK_MAX_DIMS] = {};
  int64_t span = 0;
  for (int n = 0; n < t->ndim; n++) {
    int k = -1;
    for (int i = 0; i < t->ndim; i++)
      if (!used[i] && (k < 0 || t->stride[i] < t->stride[k] || (t->stride[i] == t->stride[k] && t->shape[i] < t->shape[k]))) k = i;
    used[k] = true;
    if (t->shape[k] <= 1) continue;
    if (t->stride[k] <= span) return false;
    span += (t->shape[k] - 1) * t->stride[k];
  }
  return true;
}

inline int fill_cache8(Cache8* c, const pk_cache8* cache, bool write) {
  PK_REQUIRE(cache != nullptr, "cache is null");
  const pk_tensor *codes = cache->codes, *scales = cache->scales, *recent = cache->recent;
  PK_REQUIRE(codes != nullptr && codes->data != nullptr, "codes is null");
  PK_REQUIRE(codes->dtype == PK_I8 || codes->dtype == PK_E4M3, "codes has dtype tag %d, expected i8 or e4m3", codes->dtype);
  PK_REQUIRE(codes->ndim == 5 && codes->shape[3] == 2 && codes->shape[4] == 128 && codes->shape[2] <= (1LL << 31) - 256, "codes must be [bs,H,cap,2,128]");
  PK_CHECK_TENSOR(scales, PK_F32, 4);
  PK_CHECK_TENSOR(recent, PK_BF16, 5);
  const int64_t bs = codes->shape[0], H = codes->shape[1], cap = codes->shape[2], block = cache->block;
  PK_REQUIRE(block == 16 || block == 32 || block == 64 || block == 128, "block must be 16, 32, 64 or 128");
  PK_REQUIRE(bs < 65536 && H >= 1 && H < 65536, "sizes out of range");
  PK_REQUIRE(codes->stride[4] == 1 && aligned16(codes->data), "codes needs a unit inner stride and 16-byte alignment");
  for (int i = 0; i < 4; i++) PK_REQUIRE(codes->shape[i] <= 1 || (codes->stride[i] % 16 == 0 && codes->stride[i] >= 0), "the strides of codes must be multiples of 16");
  PK_REQUIRE(scales->shape[0] == bs && scales->shape[1] == H && scales->shape[2] == (cap + block - 1) / block && scales->shape[3] == 2, "scales must be f32 [bs,H,ceil(cap/block),2]");
  for (int i = 0; i < 4; i++) PK_REQUIRE(scales->shape[i] <= 1 || scales->stride[i] >= 0, "the strides of scales must not be negative");
  PK_REQUIRE(recent->shape[0] == bs && recent->shape[1] == H && recent->shape[3] == 2 && recent->shape[4] == 128, "recent must be bf16 [bs,H,R,2,128]");
  PK_REQUIRE(recent->shape[2] >= block && recent->shape[2] % block == 0 && recent->shape[2] < (1 << 24), "the places of recent must be a multiple of block, at least one block");
  PK_REQUIRE(row_tensor(recent), "recent needs a unit inner stride, other strides that are multiples of 8, and 16-byte alignment");
  if (write) PK_REQUIRE(apart(codes) && apart(scales) && apart(recent), "codes, scales and recent must not share memory within themselves");
  c->codes = (uint8_t*)codes->data, c->c_b = codes->stride[0], c->c_h = codes->stride[1], c->c_l = codes->stride[2], c->c_kv = codes->stride[3];
  c->scales = (float*)scales->data, c->s_b = scales->stride[0], c->s_h = scales->stride[1], c->s_j = scales->stride[2], c->s_kv = scales->stride[3];
  c->recent = (uint16_t*)recent->data, c->r_b = recent->stride[0], c->r_h = recent->stride[1], c->r_l = recent->stride[2], c->r_kv = recent->stride[3];
  c->cap = cap, c->R = (int)recent->shape[2], c->H = (int)H;
  c->shift = block == 16 ? 4 : block == 32 ? 5 : block == 64 ? 6 : 7;
  return PK_OK;
}

#ifdef __CUDACC__
// e4m3 x2 -> two floats, exactly
__device__ __forceinline__ float2 e4m3_floats(uint32_t two) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)two));
  float2 f;
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.f32.f16 %0, a;\n\tcvt.f32.f16 %1, b;\n\t}" : "=f"(f.x), "=f"(f.y) : "r"(h));
  return f;
}
// byte i of four whole numbers as a float: 2^23 + (code + 128) is a float whose last bits are the biased code
__device__ __forceinline__ float i8_float(uint32_t biased, int i) { return __uint_as_float(__byte_perm(biased, 0x4b000000u, 0x7540 + i)) - 8388736.0f; }
__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return (uint32_t)lo | (uint32_t)hi << 16;
}
// Codes of values whose largest magnitude is amax:  y M / amax to the nearest, ties to the even one, M = 127 (e4m3: 448), as 32-bit arithmetic gives it from (y M / u) / (amax / u) with a power of two
// u = 128 (512), which keeps the product from overflowing (amax / u is exact where amax has 16 bits; one of 32 bits has to be above 2^-119 or zero).  A division per value took two thirds of the kernels' instructions.
constexpr float CODE_MAGIC = 12582912.0f;   // 1.5 2^23: a sum with it ends in the whole number that the other is rounded to
__device__ __forceinline__ uint32_t code_bytes(const uint32_t* n) { return __byte_perm(__byte_perm(n[0], n[1], 0x0040), __byte_perm(n[2], n[3], 0x0040), 0x5410); }
template <bool E4M3>
__device__ __forceinline__ uint32_t code_pack(const float* q) {
  if (E4M3) return pack_e4m3(q[0], q[1], q[2], q[3]);
  uint32_t n[4];
#pragma unroll
  for (int e = 0; e < 4; e++) n[e] = __float_as_uint(q[e] + CODE_MAGIC);
  return code_bytes(n);
}
template <bool E4M3>
struct CodeScale {
  static constexpr float MOST = E4M3 ? 448.0f : 127.0f, U = E4M3 ? 512.0f : 128.0f;
  float unit;
  bool plain;   // factors are finite
  __device__ __forceinline__ explicit CodeScale(float amax) : unit(amax == 0.0f ? 1.0f : amax * (1.0f / U)), plain(amax > 1e-30f) {}
  __device__ __forceinline__ float quotient(float y) const { return (y * (MOST / U)) / unit; }
  __device__ __forceinline__ uint2 divided(const float (&y)[8]) const {
    float q[8];
#pragma unroll
    for (int i = 0; i < 8; i++) q[i] = quotient(y[i]);
    return make_uint2(code_pack<E4M3>(q), code_pack<E4M3>(q + 4));
  }
};
// Of values and a maximum of 16 bits: one Newton step.  y' = y M / u is exact, q1 = y' r with r near 1 / unit, rem = y' - q1 unit is exact (8 bits), and q1 + rem r is within 2^-44 of the quotient before
// its rounding: a tie, which is a number of nine bits, comes out as it is, and no other quotient is nearer to one than 2^-17 of itself.  Ties are a matter of the maximum: 128, 192, 160 times a power
// of two have many, so that a form with an exception for them took it for a third of all groups.
template <bool E4M3>
struct Coder16 : CodeScale<E4M3> {
  float r;
  __device__ __forceinline__ explicit Coder16(float amax) : CodeScale<E4M3>(amax) { asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(this->unit)); }
  __device__ __forceinline__ uint2 operator()(const float (&y)[8]) const {
    float q[8];
#pragma unroll
    for (int i = 0; i < 8; i += 2) {   // two values an instruction
      asm("{\n\t.reg .b64 y, q, e, r, u, m;\n\tmov.b64 y, {%2, %3};\n\tmov.b64 r, {%4, %4};\n\tmov.b64 u, {%5, %5};\n\tmov.b64 m, {%6, %6};\n\t"
          "mul.rn.f32x2 y, y, m;\n\tmul.rn.f32x2 q, y, r;\n\tfma.rn.f32x2 e, q, u, y;\n\tfma.rn.f32x2 q, e, r, q;\n\tmov.b64 {%0, %1}, q;\n\t}"
          : "=f"(q[i]), "=f"(q[i + 1])
          : "f"(y[i]), "f"(y[i + 1]), "f"(r), "f"(-this->unit), "f"(CodeScale<E4M3>::MOST / CodeScale<E4M3>::U));
    }
    return make_uint2(code_pack<E4M3>(q), code_pack<E4M3>(q + 4));
  }
};
// Whole numbers of values of 32 bits: each is multiplied by a factor that is surely above M / amax and by one that is surely below: where both round to the same code that is the code, whatever the last
// bits.  Others, one group of eight values in some hundred, are divided.
struct Coder32 : CodeScale<false> {
  float above, below;
  __device__ __forceinline__ explicit Coder32(float amax) : CodeScale<false>(amax) {
    const float f = MOST / amax;
    above = plain ? f * (1.0f + 0x1p-21f) : INFINITY, below = plain ? f * (1.0f - 0x1p-21f) : 0.0f;   // f is off by 2^-24 of itself, this product too; the quotient is off by 2^-23
  }
  __device__ __forceinline__ uint2 operator()(const float (&y)[8]) const {
    uint32_t n[8], differ = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      n[i] = __float_as_uint(__fmaf_rn(y[i], above, CODE_MAGIC));
      differ |= n[i] ^ __float_as_uint(__fmaf_rn(y[i], below, CODE_MAGIC));
    }
    return differ ? divided(y) : make_uint2(code_bytes(n), code_bytes(n + 4));
  }
};
#endif

}  // namespace pk
