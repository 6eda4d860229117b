// Attention of the drafted tokens of a sequence - a tree, given by a mask - over the cache and over the drafts themselves, and
// attention over listed blocks of the cache.  o = sum_j p_j v_j / sum_j p_j, p_j = 2^(s_j - max s), s_j = scale * log2(e) * q.k_j,
// over the rows that the query sees; a query that sees none gets zeros.
#include "common.cuh"

namespace pk {
namespace {

struct AttendParams {
  const uint16_t* q;
  int64_t q_b, q_t, q_h;
  const uint16_t *k, *v;
  int64_t k_b, k_h, k_l, v_b, v_h, v_l, cap;
  const uint16_t *dk, *dv;       // drafts
  int64_t dk_b, dk_t, dk_h, dv_b, dv_t, dv_h;
  const uint8_t* mask;
  int64_t m_b, m_t, m_j;
  const int32_t* blocks;         // [bs][T][H][n], or null: the tree's form
  int n, block;
  const int32_t* lengths;
  int T, H, G;
  float scale_log2;
  uint16_t* out;
  float* lse;
};

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
    const float M = fmaxf(m, s), f = m == -INFINITY ? 0.0f : exp2f(m - M), w = M == -INFINITY ? 0.0f : exp2f(s - M);
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

inline bool aligned16(const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15) == 0; }
// rows of 128 bf16 that 16-byte copies can read: unit inner stride, the other strides a multiple of 8
bool row_tensor(const pk_tensor* x) {
  if (x->stride[x->ndim - 1] != 1 || !aligned16(x->data)) return false;
  for (int i = 0; i + 1 < x->ndim; i++)
    if (x->shape[i] > 1 && (x->stride[i] % 8 || x->stride[i] < 0)) return false;
  return true;
}

// What both entry points share: queries, cache, lengths, output.
int fill_attend(AttendParams* p, const pk_tensor* queries, const pk_tensor* keys, const pk_tensor* values, const pk_tensor* lengths,
                float scale, const pk_tensor* out, const pk_tensor* lse) {
  PK_CHECK_TENSOR(queries, PK_BF16, 4);
  PK_CHECK_TENSOR(keys, PK_BF16, 4);
  PK_CHECK_TENSOR(values, PK_BF16, 4);
  PK_CHECK_TENSOR(lengths, PK_I32, 1);
  PK_CHECK_TENSOR(out, PK_BF16, 4);
  const int64_t bs = queries->shape[0], T = queries->shape[1], Hq = queries->shape[2], H = keys->shape[1];
  PK_REQUIRE(queries->shape[3] == 128, "queries must be bf16 [bs,T,Hq,128]");
  PK_REQUIRE(keys->shape[0] == bs && keys->shape[3] == 128 && keys->shape[2] < (1LL << 31), "keys must be bf16 [bs,H,cap,128]");
  for (int i = 0; i < 4; i++) PK_REQUIRE(values->shape[i] == keys->shape[i], "values must have the shape of keys");
  PK_REQUIRE(H >= 1 && Hq % H == 0 && Hq >= H && Hq / H <= 128, "the query heads must be a multiple of the KV heads, at most 128 of them each");
  PK_REQUIRE(row_tensor(queries) && row_tensor(keys) && row_tensor(values),
             "queries, keys and values need a unit inner stride, other strides that are multiples of 8, and 16-byte alignment");
  PK_REQUIRE(lengths->shape[0] == bs && is_contig(lengths), "lengths must be contiguous i32 [bs]");
  for (int i = 0; i < 4; i++) PK_REQUIRE(out->shape[i] == queries->shape[i], "out must have the shape of queries");
  PK_REQUIRE(is_contig(out) && aligned16(out->data), "out must be contiguous and 16-byte aligned");
  if (lse) {
    PK_CHECK_TENSOR(lse, PK_F32, 3);
    PK_REQUIRE(is_contig(lse) && lse->shape[0] == bs && lse->shape[1] == T && lse->shape[2] == Hq, "lse must be contiguous f32 [bs,T,Hq]");
    p->lse = (float*)lse->data;
  }
  PK_REQUIRE(bs < 65536 && bs * T * Hq < (1LL << 31), "sizes out of range");
  p->q = (const uint16_t*)queries->data, p->q_b = queries->stride[0], p->q_t = queries->stride[1], p->q_h = queries->stride[2];
  p->k = (const uint16_t*)keys->data, p->k_b = keys->stride[0], p->k_h = keys->stride[1], p->k_l = keys->stride[2];
  p->v = (const uint16_t*)values->data, p->v_b = values->stride[0], p->v_h = values->stride[1], p->v_l = values->stride[2];
  p->cap = keys->shape[2], p->lengths = (const int32_t*)lengths->data;
  p->T = (int)T, p->H = (int)H, p->G = (int)(Hq / H);
  p->scale_log2 = scale * 1.4426950408889634f;
  p->out = (uint16_t*)out->data;
  return PK_OK;
}

int launch_attend(const AttendParams& p, int64_t bs, const char* what, cudaStream_t st) {
  const int64_t rows = bs * p.T * p.H * p.G;
  if (rows == 0) return PK_OK;
  StageTimer timer(ST_ATTENTION, st);
  launch_chain(attend_kernel, dim3((unsigned)((rows + 3) / 4)), dim3(128), 0, st, p, rows);
  return check_launch(what);
}

}  // namespace
}  // namespace pk

using namespace pk;

extern "C" int64_t pk_tree_attention_workspace_bytes(int64_t, int64_t, int64_t, int64_t, int64_t) { return 256; }

extern "C" int pk_tree_attention(const pk_tensor* queries, const pk_tensor* keys, const pk_tensor* values, const pk_tensor* draft_keys,
                                 const pk_tensor* draft_values, const pk_tensor* tree_mask, const pk_tensor* lengths, float scale,
                                 const pk_tensor* out, const pk_tensor* lse, void*, int64_t, void* stream) {
  AttendParams p = {};
  if (const int rc = fill_attend(&p, queries, keys, values, lengths, scale, out, lse)) return rc;
  PK_CHECK_TENSOR(draft_keys, PK_BF16, 4);
  PK_CHECK_TENSOR(draft_values, PK_BF16, 4);
  PK_CHECK_TENSOR(tree_mask, PK_U8, 3);
  const int64_t bs = queries->shape[0];
  PK_REQUIRE(p.T <= 256, "at most 256 drafted tokens");
  for (const pk_tensor* d : {draft_keys, draft_values}) {
    PK_REQUIRE(d->shape[0] == bs && d->shape[1] == p.T && d->shape[2] == p.H && d->shape[3] == 128, "draft_keys / draft_values must be bf16 [bs,T,H,128]");
    PK_REQUIRE(row_tensor(d), "draft_keys / draft_values need a unit inner stride, other strides that are multiples of 8, and 16-byte alignment");
  }
  PK_REQUIRE((tree_mask->shape[0] == bs || tree_mask->shape[0] == 1) && tree_mask->shape[1] == p.T && tree_mask->shape[2] == p.T,
             "tree_mask must be [1 or bs,T,T]");
  p.dk = (const uint16_t*)draft_keys->data, p.dk_b = draft_keys->stride[0], p.dk_t = draft_keys->stride[1], p.dk_h = draft_keys->stride[2];
  p.dv = (const uint16_t*)draft_values->data, p.dv_b = draft_values->stride[0], p.dv_t = draft_values->stride[1], p.dv_h = draft_values->stride[2];
  p.mask = (const uint8_t*)tree_mask->data, p.m_b = tree_mask->shape[0] == 1 ? 0 : tree_mask->stride[0], p.m_t = tree_mask->stride[1], p.m_j = tree_mask->stride[2];
  return launch_attend(p, bs, "tree_attention", (cudaStream_t)stream);
}

extern "C" int64_t pk_block_attention_workspace_bytes(int64_t, int64_t, int64_t, int64_t, int64_t, int64_t) { return 256; }

extern "C" int pk_block_attention(const pk_tensor* queries, const pk_tensor* keys, const pk_tensor* values, const pk_tensor* blocks,
                                  const pk_tensor* lengths, int64_t block, float scale, const pk_tensor* out, const pk_tensor* lse,
                                  void*, int64_t, void* stream) {
  AttendParams p = {};
  if (const int rc = fill_attend(&p, queries, keys, values, lengths, scale, out, lse)) return rc;
  PK_CHECK_TENSOR(blocks, PK_I32, 4);
  const int64_t bs = queries->shape[0];
  PK_REQUIRE(block == 16 || block == 32 || block == 64 || block == 128, "block must be 16, 32, 64 or 128");
  PK_REQUIRE(blocks->shape[0] == bs && blocks->shape[1] == p.T && blocks->shape[2] == p.H && is_contig(blocks), "blocks must be contiguous i32 [bs,T,H,n]");
  PK_REQUIRE(blocks->shape[3] * block <= (1 << 24), "too many blocks");
  p.blocks = (const int32_t*)blocks->data, p.n = (int)blocks->shape[3], p.block = (int)block;
  return launch_attend(p, bs, "block_attention", (cudaStream_t)stream);
}
