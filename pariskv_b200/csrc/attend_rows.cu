// Attention for several tokens a step, a warp per query row with plain loads: o = sum_j p_j v_j / sum_j p_j, p_j = 2^(s_j - max s),
// s_j = scale * log2(e) * q.k_j, over the rows that the query sees; a query that sees none gets zeros.  Only for caches that tensor
// maps do not take (a dimension of stride zero: one head's rows shared by several).
#include "attend.cuh"

namespace pk {
namespace {

// A warp per query row; lane L holds dims 4L .. 4L + 3.
__global__ void __launch_bounds__(128) attend_kernel(AttendParams p, int64_t rows) {
  pdl_wait();
  pdl_trigger();
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (row >= rows) return;
  const int lane = threadIdx.x & 31, Hq = p.H * p.G;
  const int hq = (int)(row % Hq), t = (int)(row / Hq % p.T), h = hq / p.G;
  const int64_t b = row / Hq / p.T;
  auto four = [&](const uint16_t* x, float* f) {
    const uint2 r = *reinterpret_cast<const uint2*>(x + 4 * lane);
    f[0] = __uint_as_float(r.x << 16), f[1] = __uint_as_float(r.x & 0xffff0000u), f[2] = __uint_as_float(r.y << 16), f[3] = __uint_as_float(r.y & 0xffff0000u);
  };
  float q[4], o[4] = {0, 0, 0, 0}, m = -INFINITY, l = 0;
  four(p.q + b * p.q_b + t * p.q_t + hq * p.q_h, q);
  auto see = [&](const uint16_t* k, const uint16_t* v) {
    float kf[4], vf[4];
    four(k, kf), four(v, vf);
    float s = q[0] * kf[0] + q[1] * kf[1] + q[2] * kf[2] + q[3] * kf[3];
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    s *= p.scale_log2;
    const float M = fmaxf(m, s), f = m == -INFINITY ? 0.0f : exp2f(m - M), w = exp2f(s - (M == -INFINITY ? 0.0f : M));   // (NaN stays)
    l = l * f + w, m = M;
#pragma unroll
    for (int i = 0; i < 4; i++) o[i] = o[i] * f + w * vf[i];
  };
  const int64_t len = min((int64_t)max(p.lengths[b], 0), p.cap);
  const uint16_t *kb = p.k + b * p.k_b + h * p.k_h, *vb = p.v + b * p.v_b + h * p.v_h;
  if (p.blocks) {
    const int64_t end = len - p.T + t + 1;
    const int32_t* ids = p.blocks + ((b * p.T + t) * p.H + h) * p.n;
    for (int i = 0; i < p.n; i++) {
      if (ids[i] < 0) continue;
      const int64_t first = (int64_t)ids[i] * p.block, stop = min(first + p.block, end);
      for (int64_t j = first; j < stop; j++) see(kb + j * p.k_l, vb + j * p.v_l);
    }
  } else {
    for (int64_t j = 0; j < len; j++) see(kb + j * p.k_l, vb + j * p.v_l);
    for (int j = 0; j < p.T; j++)
      if (p.mask[b * p.m_b + t * p.m_t + j * p.m_j])
        see(p.dk + b * p.dk_b + j * p.dk_t + h * p.dk_h, p.dv + b * p.dv_b + j * p.dv_t + h * p.dv_h);
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  uint2 w;
  w.x = f2bf(o[0] * inv) | (uint32_t)f2bf(o[1] * inv) << 16;
  w.y = f2bf(o[2] * inv) | (uint32_t)f2bf(o[3] * inv) << 16;
  *reinterpret_cast<uint2*>(p.out + row * 128 + 4 * lane) = w;
  if (p.lse && lane == 0) p.lse[row] = l == 0.0f ? -INFINITY : m + log2f(l);
}

}  // namespace

int launch_attend_rows(const AttendParams& p, int64_t bs, const char* what, cudaStream_t st) {
  const int64_t rows = bs * p.T * p.H * p.G;
  if (rows == 0) return PK_OK;
  StageTimer timer(ST_ATTENTION, st);
  launch_chain(attend_kernel, dim3((unsigned)((rows + 3) / 4)), dim3(128), 0, st, p, rows);
  return check_launch(what);
}


}  // namespace pk
