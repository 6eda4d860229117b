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
// u = 128 (512).  A division per value took two thirds of the kernels' instructions.  Instead each is multiplied by a factor that is surely above M / amax and by one that is surely below: where both round
// to the same code that is the code, whatever the last bits.  EXACT (whole numbers of values of 16 bits): the others, which are ties or next to one, go by the sign of 2 y' - (n + n') unit, y' = y M / u,
// n and n' the two codes: products of 16 bits, one rounding.  Ties are a matter of the block's largest value - 128, 192, 160 times a power of two have many - and a division took a quarter of such a block's time.
template <bool E4M3, bool EXACT>
struct Coder {
  static constexpr float MOST = E4M3 ? 448.0f : 127.0f, U = E4M3 ? 512.0f : 128.0f;
  float unit, above, below;
  bool plain;
  __device__ __forceinline__ explicit Coder(float amax) {
    unit = amax == 0.0f ? 1.0f : __fmul_rn(amax, 1.0f / U);
    const float f = __fdiv_rn(MOST, amax);
    plain = amax > 1e-30f;   // (else the factor might be infinite)
    above = plain ? f * (1.0f + 0x1p-21f) : INFINITY, below = plain ? f * (1.0f - 0x1p-21f) : 0.0f;   // f is off by 2^-24 of itself, this product too; the quotient is off by 2^-23
  }
  __device__ __forceinline__ float quotient(float y) const { return __fdiv_rn(__fmul_rn(y, MOST / U), unit); }
  static __device__ __forceinline__ uint32_t bytes(const uint32_t* n) { return __byte_perm(__byte_perm(n[0], n[1], 0x0040), __byte_perm(n[2], n[3], 0x0040), 0x5410); }
  __device__ __forceinline__ uint2 operator()(const float (&y)[8]) const {
    uint32_t a[2], differ = 0;
    if (E4M3) {
#pragma unroll
      for (int i = 0; i < 2; i++) {
        a[i] = pack_e4m3(y[4 * i] * above, y[4 * i + 1] * above, y[4 * i + 2] * above, y[4 * i + 3] * above);
        differ |= a[i] ^ pack_e4m3(y[4 * i] * below, y[4 * i + 1] * below, y[4 * i + 2] * below, y[4 * i + 3] * below);
      }
      if (differ) {
#pragma unroll
        for (int i = 0; i < 2; i++) a[i] = pack_e4m3(quotient(y[4 * i]), quotient(y[4 * i + 1]), quotient(y[4 * i + 2]), quotient(y[4 * i + 3]));
      }
    } else {
      uint32_t n[8];
#pragma unroll
      for (int i = 0; i < 8; i++) {   // the sum with 1.5 2^23 ends in the whole number
        n[i] = __float_as_uint(__fmaf_rn(y[i], above, 12582912.0f));
        differ |= n[i] ^ __float_as_uint(__fmaf_rn(y[i], below, 12582912.0f));
      }
      if (differ) {
        if (EXACT && plain) {
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const uint32_t m = __float_as_uint(__fmaf_rn(y[i], below, 12582912.0f));
            const float both = (__uint_as_float(n[i]) - 12582912.0f) + (__uint_as_float(m) - 12582912.0f);
            const float d = __fmaf_rn(2.0f, __fmul_rn(y[i], MOST / U), -both * unit) * (y[i] < 0.0f ? -1.0f : 1.0f);   // above zero: n, which is the one of the larger magnitude
            n[i] = d > 0.0f || (d == 0.0f && (n[i] & 1) == 0) ? n[i] : m;
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; i++) n[i] = (uint32_t)__float2int_rn(quotient(y[i]));
        }
      }
      a[0] = bytes(n), a[1] = bytes(n + 4);
    }
    return make_uint2(a[0], a[1]);
  }
};
#endif

}  // namespace pk
