// Block bounds of the keys of a cache, and the selection of blocks by them.
//   bounds[j] = (lo, hi): smallest and largest value per channel over the rows of block j
//   score_j   = sum_d sum_g max(q_gd lo_jd, q_gd hi_jd), no less than the sum over the group's query heads g of q_g.k for any key k of the
//               block;  with P_d = sum_g max(q_gd, 0) and N_d = sum_g min(q_gd, 0) it is sum_d P_d hi_jd + N_d lo_jd: one pass over the
//               bounds whatever the number of query heads.
// Sums in 64 bits, rounded once to 32: the choice does not depend on their order.
#include "attend.cuh"

namespace pk {
namespace {

struct BoundsParams {
  const uint16_t* k;
  int64_t k_b, k_h, k_l, cap;
  const int32_t* lengths;
  uint16_t* out;          // [..][NB][2][128] by strides
  int64_t o_b, o_h, o_j;
  int H, block, n_new;    // n_new < 0: all blocks
};

// A warp per block of keys; lane L holds channels 4L .. 4L + 3.
__global__ void __launch_bounds__(128) block_bounds_kernel(BoundsParams p, int64_t per_head) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, h = blockIdx.y, b = blockIdx.z;
  const int64_t len = p.lengths ? min((int64_t)max(p.lengths[b], 0), p.cap) : p.cap;
  const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (at >= per_head) return;
  const int64_t j = at + (p.n_new < 0 ? 0 : max((int64_t)0, len - p.n_new) / p.block), first = j * p.block, end = min(first + p.block, len);
  if (first >= end) return;
  const uint16_t* k = p.k + b * p.k_b + h * p.k_h + 4 * lane;
  const __nv_bfloat162 *row = reinterpret_cast<const __nv_bfloat162*>(k + first * p.k_l);
  __nv_bfloat162 lo[2] = {row[0], row[1]}, hi[2] = {row[0], row[1]};
  for (int64_t r = first + 1; r < end; r++) {
    row = reinterpret_cast<const __nv_bfloat162*>(k + r * p.k_l);
#pragma unroll
    for (int i = 0; i < 2; i++) lo[i] = __hmin2_nan(lo[i], row[i]), hi[i] = __hmax2_nan(hi[i], row[i]);
  }
  __nv_bfloat162* o = reinterpret_cast<__nv_bfloat162*>(p.out + b * p.o_b + h * p.o_h + j * p.o_j + 4 * lane);
  o[0] = lo[0], o[1] = lo[1], o[64] = hi[0], o[65] = hi[1];
}

struct SelectParams {
  const uint16_t* q;
  int64_t q_b, q_t, q_h;
  const uint16_t* bounds;
  int64_t o_b, o_h, o_j, nb;
  const int32_t* lengths;
  int T, H, G, n, block, sink, local;
  uint32_t* keys;      // [rows][nb] ordered keys of the scores
  int32_t* ids;        // [rows][n]
};

constexpr uint32_t FORCED = 0xffffffffu, NOT_A_NUMBER = 0xfffffffeu;

// Blocks that row (b, t) sees.
__device__ __forceinline__ int64_t visible_blocks(const SelectParams& p, int64_t b, int t) {
  const int64_t pos = min((int64_t)p.lengths[b], p.nb * p.block) - p.T + t;
  return pos < 0 ? 0 : pos / p.block + 1;
}

// A warp per (row, block of keys).
__global__ void __launch_bounds__(128) block_score_kernel(SelectParams p) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  const int64_t row = blockIdx.y, h = row % p.H, t = row / p.H % p.T, b = row / p.H / p.T;
  const int64_t seen = visible_blocks(p, b, (int)t), j = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (j >= seen) return;
  double s = 0.0;
  const uint16_t* bd = p.bounds + b * p.o_b + h * p.o_h + j * p.o_j;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    double up = 0.0, down = 0.0;
    for (int g = 0; g < p.G; g++) {
      const double x = bf2f(p.q[b * p.q_b + t * p.q_t + (h * p.G + g) * p.q_h + 4 * lane + i]);
      if (x < 0) down += x;
      else up += x;
    }
    // (no products of a zero with an infinite bound)
    s += !(up == 0) ? up * bf2f(bd[128 + 4 * lane + i]) : 0.0;
    s += !(down == 0) ? down * bf2f(bd[4 * lane + i]) : 0.0;
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
  if (lane == 0) {
    const float f = (float)s + 0.0f;   // (one zero)
    p.keys[row * p.nb + j] = j < p.sink || j >= seen - p.local ? FORCED : f != f ? NOT_A_NUMBER : ord_key(f);
  }
}

// A block per row: the n-th largest key bit by bit, then the chosen ones in order.
__global__ void __launch_bounds__(256) block_pick_kernel(SelectParams p) {
  pdl_wait();
  pdl_trigger();
  const int64_t row = blockIdx.x, t = row / p.H % p.T, b = row / p.H / p.T;
  const int64_t seen = visible_blocks(p, b, (int)t);
  const uint32_t* keys = p.keys + row * p.nb;
  int32_t* ids = p.ids + row * p.n;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  __shared__ int s_count[8], s_ties[8];
  const int n = (int)min((int64_t)p.n, seen);
  for (int i = n + tid; i < p.n; i += 256) ids[i] = -1;
  uint32_t cut = 0;
  int above = 0;
  auto count = [&](uint32_t least) {   // keys >= least
    int c = 0;
    for (int64_t j = tid; j < seen; j += 256) c += keys[j] >= least;
    c = __reduce_add_sync(0xffffffffu, c);
    __syncthreads();
    if (lane == 0) s_count[warp] = c;
    __syncthreads();
    int total = 0;
    for (int w = 0; w < 8; w++) total += s_count[w];
    return total;
  };
  for (int bit = 31; bit >= 0; bit--)
    if (count(cut | 1u << bit) >= n) cut |= 1u << bit;
  above = cut == 0xffffffffu ? 0 : count(cut + 1);
  int placed = 0, ties_seen = 0;
  for (int64_t j0 = 0; j0 < seen; j0 += 256) {
    const int64_t j = j0 + tid;
    const uint32_t k = j < seen ? keys[j] : 0;
    const bool tie = j < seen && k == cut;
    const unsigned tie_bits = __ballot_sync(0xffffffffu, tie);
    __syncthreads();
    if (lane == 0) s_ties[warp] = __popc(tie_bits);
    __syncthreads();
    int before = ties_seen, all = 0;
    for (int w = 0; w < 8; w++) before += w < warp ? s_ties[w] : 0, all += s_ties[w];
    const bool take = j < seen && (k > cut || (tie && before + __popc(tie_bits & ((1u << lane) - 1)) < n - above));
    ties_seen += all;
    const unsigned bits = __ballot_sync(0xffffffffu, take);
    if (lane == 0) s_count[warp] = __popc(bits);
    __syncthreads();
    int at = placed;
    for (int w = 0; w < 8; w++) at += w < warp ? s_count[w] : 0, placed += s_count[w];
    if (take) ids[at + __popc(bits & ((1u << lane) - 1))] = (int32_t)j;
  }
}

int check_bounds(const pk_tensor* bounds) {
  PK_CHECK_TENSOR(bounds, PK_BF16, 5);
  PK_REQUIRE(bounds->shape[3] == 2 && bounds->shape[4] == 128, "bounds must be bf16 [bs,H,blocks,2,128]");
  PK_REQUIRE(row_tensor(bounds) && bounds->stride[3] == 128, "the two rows of a block's bounds must lie next to each other, 16-byte aligned, the other strides multiples of 8");
  return PK_OK;
}
bool block_size_ok(int64_t block) { return block == 16 || block == 32 || block == 64 || block == 128; }

}  // namespace
}  // namespace pk

using namespace pk;

extern "C" int pk_block_bounds(const pk_tensor* keys, const pk_tensor* lengths, int64_t block, int64_t n_new, const pk_tensor* bounds, void* stream) {
  PK_CHECK_TENSOR(keys, PK_BF16, 4);
  if (const int rc = check_bounds(bounds)) return rc;
  const int64_t bs = keys->shape[0], H = keys->shape[1], cap = keys->shape[2];
  PK_REQUIRE(block_size_ok(block), "block must be 16, 32, 64 or 128");
  PK_REQUIRE(keys->shape[3] == 128 && cap < (1LL << 31) && row_tensor(keys), "keys must be bf16 [bs,H,cap,128] with a unit inner stride, other strides that are multiples of 8, and 16-byte alignment");
  PK_REQUIRE(bounds->shape[0] == bs && bounds->shape[1] == H && bounds->shape[2] == (cap + block - 1) / block, "bounds must be bf16 [bs,H,ceil(cap/block),2,128]");
  PK_REQUIRE(n_new >= -1 && n_new < (1LL << 31), "n_new must be a number of rows, or -1 for all blocks");
  BoundsParams p = {};
  if (lengths) {
    PK_CHECK_TENSOR(lengths, PK_I32, 1);
    PK_REQUIRE(lengths->shape[0] == bs && is_contig(lengths), "lengths must be contiguous i32 [bs]");
    p.lengths = (const int32_t*)lengths->data;
  }
  PK_REQUIRE(bs < 65536 && H < 65536, "sizes out of range");
  p.k = (const uint16_t*)keys->data, p.k_b = keys->stride[0], p.k_h = keys->stride[1], p.k_l = keys->stride[2], p.cap = cap;
  p.out = (uint16_t*)bounds->data, p.o_b = bounds->stride[0], p.o_h = bounds->stride[1], p.o_j = bounds->stride[2];
  p.H = (int)H, p.block = (int)block, p.n_new = (int)n_new;
  int64_t per_head = bounds->shape[2];
  if (n_new >= 0) per_head = n_new == 0 ? 0 : (n_new + block - 2) / block + 1 < per_head ? (n_new + block - 2) / block + 1 : per_head;
  if (bs * H * per_head == 0) return PK_OK;
  StageTimer timer(ST_ENCODE, (cudaStream_t)stream);
  launch_chain(block_bounds_kernel, dim3((unsigned)((per_head + 3) / 4), (unsigned)H, (unsigned)bs), dim3(128), 0, (cudaStream_t)stream, p, per_head);
  return check_launch("block_bounds");
}

extern "C" int64_t pk_select_blocks_workspace_bytes(int64_t bs, int64_t T, int64_t H, int64_t n_blocks) { return bs * T * H * n_blocks * 4 + 256; }

extern "C" int pk_select_blocks(const pk_tensor* queries, const pk_tensor* bounds, const pk_tensor* lengths, int64_t block, int64_t sink_blocks,
                                int64_t local_blocks, const pk_tensor* blocks, void* workspace, int64_t workspace_bytes, void* stream) {
  PK_CHECK_TENSOR(queries, PK_BF16, 4);
  if (const int rc = check_bounds(bounds)) return rc;
  PK_CHECK_TENSOR(lengths, PK_I32, 1);
  PK_CHECK_TENSOR(blocks, PK_I32, 4);
  const int64_t bs = queries->shape[0], T = queries->shape[1], Hq = queries->shape[2], H = bounds->shape[1], nb = bounds->shape[2], n = blocks->shape[3];
  PK_REQUIRE(block_size_ok(block), "block must be 16, 32, 64 or 128");
  PK_REQUIRE(queries->shape[3] == 128 && row_tensor(queries), "queries must be bf16 [bs,T,Hq,128] with a unit inner stride, other strides that are multiples of 8, and 16-byte alignment");
  PK_REQUIRE(bounds->shape[0] == bs && H >= 1 && Hq >= H && Hq % H == 0, "the query heads must be a multiple of the KV heads of bounds");
  PK_REQUIRE(lengths->shape[0] == bs && is_contig(lengths), "lengths must be contiguous i32 [bs]");
  PK_REQUIRE(blocks->shape[0] == bs && blocks->shape[1] == T && blocks->shape[2] == H && is_contig(blocks), "blocks must be contiguous i32 [bs,T,H,n]");
  PK_REQUIRE(sink_blocks >= 0 && local_blocks >= 1 && sink_blocks + local_blocks <= n, "at least one local block, and no more sink and local blocks than are selected");
  PK_REQUIRE(nb * block < (1LL << 31) && n < (1LL << 24) && bs * T * H < 65536LL * 32768, "sizes out of range");
  if (bs * T * H == 0) return PK_OK;
  if (!workspace || workspace_bytes < pk_select_blocks_workspace_bytes(bs, T, H, nb)) return fail(PK_ERR_WORKSPACE, "select_blocks: workspace missing or too small");
  SelectParams p = {};
  p.q = (const uint16_t*)queries->data, p.q_b = queries->stride[0], p.q_t = queries->stride[1], p.q_h = queries->stride[2];
  p.bounds = (const uint16_t*)bounds->data, p.o_b = bounds->stride[0], p.o_h = bounds->stride[1], p.o_j = bounds->stride[2], p.nb = nb;
  p.lengths = (const int32_t*)lengths->data, p.T = (int)T, p.H = (int)H, p.G = (int)(Hq / H), p.n = (int)n, p.block = (int)block;
  p.sink = (int)sink_blocks, p.local = (int)local_blocks, p.keys = (uint32_t*)workspace, p.ids = (int32_t*)blocks->data;
  const int64_t rows = bs * T * H;
  PK_REQUIRE(rows < 65536, "at most 65535 rows (batch x tokens x KV heads)");
  StageTimer timer(ST_RANK, (cudaStream_t)stream);
  if (nb > 0) launch_chain(block_score_kernel, dim3((unsigned)((nb + 3) / 4), (unsigned)rows), dim3(128), 0, (cudaStream_t)stream, p);
  launch_chain(block_pick_kernel, dim3((unsigned)rows), dim3(256), 0, (cudaStream_t)stream, p);
  return check_launch("select_blocks", nb > 0 ? 2 : 1);
}
