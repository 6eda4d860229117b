// What the attention entry points for several tokens a step share: arguments and their checks.
#pragma once
#include "common.cuh"

namespace pk {

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


inline bool aligned16(const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15) == 0; }
// rows of 128 bf16 that 16-byte copies can read: unit inner stride, the other strides a multiple of 8
inline bool row_tensor(const pk_tensor* x) {
  if (x->stride[x->ndim - 1] != 1 || !aligned16(x->data)) return false;
  for (int i = 0; i + 1 < x->ndim; i++)
    if (x->shape[i] > 1 && (x->stride[i] % 8 || x->stride[i] < 0)) return false;
  return true;
}

// What both entry points share: queries, cache, lengths, output.
inline int fill_attend(AttendParams* p, const pk_tensor* queries, const pk_tensor* keys, const pk_tensor* values, const pk_tensor* lengths,
                float scale, const pk_tensor* out, const pk_tensor* lse) {
  PK_CHECK_TENSOR(queries, PK_BF16, 4);
  PK_CHECK_TENSOR(keys, PK_BF16, 4);
  PK_CHECK_TENSOR(values, PK_BF16, 4);
  PK_CHECK_TENSOR(lengths, PK_I32, 1);
  PK_CHECK_TENSOR(out, PK_BF16, 4);
  const int64_t bs = queries->shape[0], T = queries->shape[1], Hq = queries->shape[2], H = keys->shape[1];
  PK_REQUIRE(queries->shape[3] == 128, "queries must be bf16 [bs,T,Hq,128]");
  PK_REQUIRE(keys->shape[0] == bs && keys->shape[3] == 128 && keys->shape[2] <= (1LL << 31) - 128, "keys must be bf16 [bs,H,cap,128]");
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
  PK_REQUIRE(scale > 0.0f && p->scale_log2 <= 3.4e38f, "scale must be positive, and finite as a factor of log2 e");
  return PK_OK;
}

// One warp per query row, plain loads: for the strides that tensor maps do not take.
int launch_attend_rows(const AttendParams& p, int64_t bs, const char* what, cudaStream_t st);
// Drafted tokens of up to 16 query rows per KV head, listed blocks (attend_few.cu); workspace: attend_few_workspace() bytes.
int launch_attend_few(const AttendParams& p, int64_t bs, void* workspace, const char* what, cudaStream_t st);
int64_t attend_few_workspace();

}  // namespace pk
