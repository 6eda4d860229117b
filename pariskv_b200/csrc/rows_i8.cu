// Rows of 16-bit values as 8-bit whole numbers with a scale per row: of a residual stream through its norm, of a gated activation, or of the rows themselves.
//   y = bf16(a + r) rstd w  |  silu(g) u  |  x,      scale = max |y| / 127,   code = y 127 / max |y| to the nearest
// A block per row; the row stays in registers through both reductions.
#include <type_traits>

#include "cache8.cuh"

namespace pk {
namespace {

enum { NORM, PLAIN, GATED };

struct RowParams {
  const uint16_t *a, *r, *w;
  int64_t a_s, r_s, h_s, c_s;   // strides of the rows
  uint16_t* h;
  uint8_t* codes;
  float* scales;
  int n;
  double eps, one_n;   // one_n: 1 / n
};

__device__ __forceinline__ float part(uint32_t w, int i) { return __uint_as_float(i ? w & 0xffff0000u : w << 16); }

// 1 / sqrt(x) to the last bits of 64, by Newton's iteration from 32 bits: every thread computes it, and a division and a root of 64 bits are some hundred instructions.
__device__ __forceinline__ double inverse_root(double x) {
  if (!(x > 1e-30 && x < 1e30)) return 1.0 / sqrt(x);
  double r = rsqrtf((float)x);
#pragma unroll
  for (int i = 0; i < 2; i++) r = fma(0.5 * r, fma(-x * r, r, 1.0), r);
  return r;
}

template <int MODE, int THREADS, int N>   // N groups of 8 values a thread
__global__ void __launch_bounds__(THREADS) rows_i8_kernel(const __grid_constant__ RowParams p) {
  __shared__ double s_sum[THREADS / 32];
  __shared__ uint32_t s_max[THREADS / 32];
  pdl_wait();
  pdl_trigger();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t row = blockIdx.x;
  float y[N][8];
  if (MODE == NORM) {
    constexpr int M = N < 4 ? N : 4;   // groups whose loads are all under way before the first is used
    double ss = 0.0;
#pragma unroll
    for (int k0 = 0; k0 < N; k0 += M) {
      uint4 h[M], rv[M];
#pragma unroll
      for (int k = 0; k < M; k++) {
        const int i = ((k0 + k) * THREADS + tid) * 8;
        h[k] = i < p.n ? *reinterpret_cast<const uint4*>(p.a + row * p.a_s + i) : make_uint4(0, 0, 0, 0);
      }
      if (p.r) {
#pragma unroll
        for (int k = 0; k < M; k++) {
          const int i = ((k0 + k) * THREADS + tid) * 8;
          rv[k] = i < p.n ? *reinterpret_cast<const uint4*>(p.r + row * p.r_s + i) : make_uint4(0, 0, 0, 0);
        }
      }
#pragma unroll
      for (int k = 0; k < M; k++) {
        const int i = ((k0 + k) * THREADS + tid) * 8;
        uint32_t hw[4] = {h[k].x, h[k].y, h[k].z, h[k].w};
        if (p.r) {
          const uint32_t rw[4] = {rv[k].x, rv[k].y, rv[k].z, rv[k].w};
#pragma unroll
          for (int e = 0; e < 4; e++) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(hw[e]) : "f"(part(hw[e], 1) + part(rw[e], 1)), "f"(part(hw[e], 0) + part(rw[e], 0)));
        }
        if (i < p.n) *reinterpret_cast<uint4*>(p.h + row * p.h_s + i) = make_uint4(hw[0], hw[1], hw[2], hw[3]);
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const float f = part(hw[e >> 1], e & 1);
          y[k0 + k][e] = f;
          // f as a double, by its bits (a conversion takes four times as long): what is below 2^-126 counts as at most that, what is not a number as 2^128 - the row's maximum tells
          const double d = __hiloint2double((int)((__float_as_uint(f) & 0x7fffffffu) >> 3) + 0x38000000, 0);
          ss = fma(d, d, ss);
        }
      }
    }
    auto row_sum = [&](double v) {
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
      if (lane == 0) s_sum[warp] = v;
      __syncthreads();
      v = 0.0;
#pragma unroll
      for (int i = 0; i < THREADS / 32; i++) v += s_sum[i];
      return v;
    };
    ss = row_sum(ss);
    if (ss < 1e-60 && p.eps < 1e-50) {   // a row of next to nothing, without an eps to speak of: by conversions after all
      ss = 0.0;
#pragma unroll 1
      for (int i = tid; i < p.n; i += THREADS) {
        const double d = bf2f(p.h[row * p.h_s + i]);
        ss = fma(d, d, ss);
      }
      __syncthreads();
      ss = row_sum(ss);
    }
    const float rstd = (float)inverse_root(fma(ss, p.one_n, p.eps));
#pragma unroll
    for (int k = 0; k < N; k++) {
      const int i = (k * THREADS + tid) * 8;
      if (i < p.n) {
        const uint4 wv = *reinterpret_cast<const uint4*>(p.w + i);
        const uint32_t ww[4] = {wv.x, wv.y, wv.z, wv.w};
#pragma unroll
        for (int e = 0; e < 8; e++) y[k][e] = __fmul_rn(__fmul_rn(y[k][e], rstd), part(ww[e >> 1], e & 1));
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < N; k++) {
      const int i = (k * THREADS + tid) * 8;
      if (i < p.n) {
        const uint4 xv = *reinterpret_cast<const uint4*>(p.a + row * p.a_s + i);
        const uint4 uv = MODE == GATED ? *reinterpret_cast<const uint4*>(p.a + row * p.a_s + p.n + i) : make_uint4(0, 0, 0, 0);
        const uint32_t xw[4] = {xv.x, xv.y, xv.z, xv.w};
#pragma unroll
        for (int e = 0; e < 8; e++) y[k][e] = part(xw[e >> 1], e & 1);
        if (MODE == GATED) {
          const uint32_t uw[4] = {uv.x, uv.y, uv.z, uv.w};
#pragma unroll
          for (int e = 0; e < 8; e++) y[k][e] = y[k][e] / (1.0f + expf(-y[k][e])) * part(uw[e >> 1], e & 1);
        }
      }
    }
  }
  uint32_t m = 0;
#pragma unroll
  for (int k = 0; k < N; k++)
    if ((k * THREADS + tid) * 8 < p.n) {
#pragma unroll
      for (int e = 0; e < 8; e++) m = max(m, __float_as_uint(y[k][e]) & 0x7fffffffu);   // (what is not a number is above infinity)
    }
  m = __reduce_max_sync(0xffffffffu, m);
  if (lane == 0) s_max[warp] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < THREADS / 32; i++) m = max(m, s_max[i]);
  const bool fine = m < 0x7f800000u;
  const float amax = __uint_as_float(m);
  const bool small = MODE != PLAIN && amax < 1e-30f;   // amax / 128 may be no number of 32 bits: the row and its maximum are multiplied by 2^64, which is exact
  if (small) {
#pragma unroll
    for (int k = 0; k < N; k++)
#pragma unroll
      for (int e = 0; e < 8; e++) y[k][e] *= 0x1p64f;
  }
  const std::conditional_t<MODE == PLAIN, Coder16<false>, Coder32> code(small ? amax * 0x1p64f : amax);
#pragma unroll
  for (int k = 0; k < N; k++) {
    const int i = (k * THREADS + tid) * 8;
    if (i < p.n) {
      uint2 o = make_uint2(0, 0);
      if (fine) o = MODE == PLAIN && !code.plain ? code.divided(y[k]) : code(y[k]);
      *reinterpret_cast<uint2*>(p.codes + row * p.c_s + i) = o;
    }
  }
  if (tid == 0) p.scales[row] = fine ? __fdiv_rn(amax, 127.0f) : NAN;
}

template <int MODE, int THREADS, int N>
void launch_as(const RowParams& p, int64_t rows, cudaStream_t st) {
  launch_chain(rows_i8_kernel<MODE, THREADS, N>, dim3((unsigned)rows), dim3(THREADS), 0, st, p);
}
// Few rows: 512 threads, a group of eight values each as far as that goes, for the shortest way through a row.  Many: two or four groups a thread, so that a block has few warps to wait for and an SM more
// blocks at different places.  B200, rows of 4096, us, 512 | 256 | 128 threads: 1000 of them 7.6 | 6.5 | 7.4, 4096 of them 27.7 | 23.2 | 22.4 (5.2 TB/s).
template <int MODE>
int launch(const RowParams& p, int64_t rows, const char* what, cudaStream_t st) {
  StageTimer timer(ST_GLUE, st);
  const bool many = rows >= 2 * sm_count();
  if (many && p.n <= 2048) launch_as<MODE, 64, 4>(p, rows, st);
  else if (rows >= 16 * sm_count() && p.n <= 4096) launch_as<MODE, 128, 4>(p, rows, st);
  else if (many && p.n <= 4096) launch_as<MODE, 256, 2>(p, rows, st);
  else if (many && p.n <= 8192) launch_as<MODE, 256, 4>(p, rows, st);
  else if (p.n <= 4096) launch_as<MODE, 512, 1>(p, rows, st);
  else if (p.n <= 8192) launch_as<MODE, 512, 2>(p, rows, st);
  else if (p.n <= 16384) launch_as<MODE, 512, 4>(p, rows, st);
  else if (p.n <= 32768) launch_as<MODE, 512, 8>(p, rows, st);
  else launch_as<MODE, 512, 16>(p, rows, st);
  return check_launch(what);
}

// rows of n values that 16-byte (codes: 8-byte) accesses reach
bool rows_ok(const pk_tensor* t, bool write) {
  return (t->shape[1] <= 1 || t->stride[1] == 1) && aligned16(t->data) && (t->shape[0] <= 1 || (t->stride[0] % 8 == 0 && t->stride[0] >= (write ? t->shape[1] : 0)));
}
int size_ok(int64_t B, int64_t n) {
  PK_REQUIRE(n >= 8 && n % 8 == 0 && n <= 65536, "the width must be a multiple of 8, at most 65536");
  PK_REQUIRE(B < (1LL << 31), "sizes out of range");
  return PK_OK;
}
int outputs_ok(const pk_tensor* codes, const pk_tensor* scales, int64_t B, int64_t n) {
  PK_CHECK_TENSOR(codes, PK_I8, 2);
  PK_CHECK_TENSOR(scales, PK_F32, 1);
  PK_REQUIRE(codes->shape[0] == B && codes->shape[1] == n && rows_ok(codes, true), "codes must be i8 [B,n], rows apart at strides that are multiples of 8, 16-byte aligned");
  PK_REQUIRE(scales->shape[0] == B && is_contig(scales), "scales must be contiguous f32 [B]");
  return PK_OK;
}

}  // namespace
}  // namespace pk

using namespace pk;

extern "C" int pk_add_rmsnorm_i8(const pk_tensor* a, const pk_tensor* residual, const pk_tensor* weight, const pk_tensor* h_out, const pk_tensor* codes, const pk_tensor* scales, double eps,
                                 void* stream) {
  PK_CHECK_TENSOR(a, PK_BF16, 2);
  PK_CHECK_TENSOR(weight, PK_BF16, 1);
  PK_CHECK_TENSOR(h_out, PK_BF16, 2);
  const int64_t B = a->shape[0], n = a->shape[1];
  if (const int rc = size_ok(B, n)) return rc;
  if (residual) {
    PK_CHECK_TENSOR(residual, PK_BF16, 2);
    PK_REQUIRE(residual->shape[0] == B && residual->shape[1] == n && rows_ok(residual, false), "residual must be bf16 [B,n], rows at strides that are multiples of 8, 16-byte aligned");
  }
  PK_REQUIRE(rows_ok(a, false), "a must have rows at strides that are multiples of 8, 16-byte aligned");
  PK_REQUIRE(h_out->shape[0] == B && h_out->shape[1] == n && rows_ok(h_out, true), "h_out must be bf16 [B,n], rows apart at strides that are multiples of 8, 16-byte aligned");
  PK_REQUIRE(weight->shape[0] == n && is_contig(weight) && aligned16(weight->data), "weight must be contiguous bf16 [n], 16-byte aligned");
  PK_REQUIRE(eps >= 0.0, "eps must not be negative");
  if (const int rc = outputs_ok(codes, scales, B, n)) return rc;
  if (B == 0) return PK_OK;
  RowParams p = {};
  p.a = (const uint16_t*)a->data, p.r = residual ? (const uint16_t*)residual->data : nullptr, p.w = (const uint16_t*)weight->data, p.h = (uint16_t*)h_out->data;
  p.codes = (uint8_t*)codes->data, p.scales = (float*)scales->data, p.n = (int)n, p.eps = eps, p.one_n = 1.0 / (double)n;
  p.a_s = a->stride[0], p.r_s = residual ? residual->stride[0] : 0, p.h_s = h_out->stride[0], p.c_s = codes->stride[0];
  return launch<NORM>(p, B, "add_rmsnorm_i8", (cudaStream_t)stream);
}

extern "C" int pk_quantize_rows_i8(const pk_tensor* x, int gated, const pk_tensor* codes, const pk_tensor* scales, void* stream) {
  PK_CHECK_TENSOR(x, PK_BF16, 2);
  const int64_t B = x->shape[0], n = gated ? x->shape[1] / 2 : x->shape[1];
  PK_REQUIRE(!gated || x->shape[1] % 2 == 0, "gated rows must be [gate, up], an even number of values");
  if (const int rc = size_ok(B, n)) return rc;
  PK_REQUIRE(rows_ok(x, false), "x must have rows at strides that are multiples of 8, 16-byte aligned");
  if (const int rc = outputs_ok(codes, scales, B, n)) return rc;
  if (B == 0) return PK_OK;
  RowParams p = {};
  p.a = (const uint16_t*)x->data, p.a_s = x->stride[0], p.codes = (uint8_t*)codes->data, p.c_s = codes->stride[0], p.scales = (float*)scales->data, p.n = (int)n;
  return gated ? launch<GATED>(p, B, "quantize_rows_i8", (cudaStream_t)stream) : launch<PLAIN>(p, B, "quantize_rows_i8", (cudaStream_t)stream);
}
