// y = x W^T for a few tokens, W of 4-bit codes c with a scale s (and an offset m) per row and group of columns:
// W = (c - 8) s, or c s + m.  Products of a group are summed before they are scaled: y = sum over groups s (sum c x) + m (sum x).
#include "common.cuh"

namespace pk {
namespace {

// A warp per (output, token).
__global__ void __launch_bounds__(128) gemv_w4_kernel(const uint8_t* w, const uint16_t* scales, const uint16_t* offsets, const uint16_t* x,
                                                      int64_t x_t, uint16_t* out, int n_out, int I, int group, int gated) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, o = blockIdx.x * 4 + (threadIdx.x >> 5), t = blockIdx.y;
  if (o >= n_out) return;
  const uint16_t* xt = x + t * x_t;
  float y[2] = {0.0f, 0.0f};
  for (int u = 0; u <= gated; u++) {
    const int64_t row = o + (int64_t)u * n_out;
    for (int i = 8 * lane; i < I; i += 256) {
      const uint32_t c = *reinterpret_cast<const uint32_t*>(w + row * (I / 2) + i / 2);
      float dot = 0.0f, sum = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const float v = bf2f(xt[i + j]), code = (float)((c >> 4 * j) & 15);
        dot += (offsets ? code : code - 8.0f) * v, sum += v;
      }
      const int64_t g = row * (I / group) + i / group;
      y[u] += bf2f(scales[g]) * dot + (offsets ? bf2f(offsets[g]) * sum : 0.0f);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) y[u] += __shfl_xor_sync(0xffffffffu, y[u], off);
  }
  if (lane == 0) out[(int64_t)t * n_out + o] = f2bf(gated ? y[0] / (1.0f + __expf(-y[0])) * y[1] : y[0]);
}

inline bool aligned16(const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15) == 0; }

}  // namespace
}  // namespace pk

using namespace pk;

extern "C" int pk_gemv_w4(const pk_tensor* weight, const pk_tensor* scales, const pk_tensor* offsets, const pk_tensor* x, const pk_tensor* out,
                          int gated, void* stream) {
  PK_CHECK_TENSOR(weight, PK_U8, 2);
  PK_CHECK_TENSOR(scales, PK_BF16, 2);
  PK_CHECK_TENSOR(x, PK_BF16, 2);
  PK_CHECK_TENSOR(out, PK_BF16, 2);
  const int64_t O = weight->shape[0], I = weight->shape[1] * 2, T = x->shape[0], groups = scales->shape[1];
  PK_REQUIRE(groups >= 1 && I % groups == 0, "scales must be bf16 [O, I / group]");
  const int64_t group = I / groups;
  PK_REQUIRE(group == 32 || group == 64 || group == 128, "the group must be 32, 64 or 128 columns");
  PK_REQUIRE(is_contig(weight) && is_contig(scales) && scales->shape[0] == O, "weight must be contiguous u8 [O,I/2], scales bf16 [O,I/group]");
  if (offsets) {
    PK_CHECK_TENSOR(offsets, PK_BF16, 2);
    PK_REQUIRE(is_contig(offsets) && offsets->shape[0] == O && offsets->shape[1] == groups, "offsets must be contiguous bf16 like scales");
  }
  PK_REQUIRE(x->shape[1] == I && x->stride[1] == 1 && (T <= 1 || (x->stride[0] >= 0 && x->stride[0] % 8 == 0)), "x must be bf16 [T,I] with a unit inner stride and a row stride that is a multiple of 8");
  PK_REQUIRE(T <= 16, "at most 16 tokens");
  PK_REQUIRE(I <= 32768 && O >= 1 && O < (1LL << 30), "at most 32768 columns");
  PK_REQUIRE(!gated || O % 2 == 0, "a gated product takes an even number of rows");
  PK_REQUIRE(is_contig(out) && out->shape[0] == T && out->shape[1] == (gated ? O / 2 : O), "out must be contiguous bf16 [T,O] (O/2 when gated)");
  PK_REQUIRE(aligned16(weight->data) && aligned16(x->data), "weight and x must be 16-byte aligned");
  if (T == 0) return PK_OK;
  const int n_out = (int)(gated ? O / 2 : O);
  StageTimer timer(ST_GEMV, (cudaStream_t)stream);
  launch_chain(gemv_w4_kernel, dim3((unsigned)((n_out + 3) / 4), (unsigned)T), dim3(128), 0, (cudaStream_t)stream, (const uint8_t*)weight->data,
               (const uint16_t*)scales->data, offsets ? (const uint16_t*)offsets->data : (const uint16_t*)nullptr, (const uint16_t*)x->data, x->stride[0],
               (uint16_t*)out->data, n_out, (int)I, (int)group, gated ? 1 : 0);
  return check_launch("gemv_w4");
}
