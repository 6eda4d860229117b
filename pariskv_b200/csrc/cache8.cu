// Rows into the cache in 8 bits and back.
//   append  scale = max |x| / 127, code = x / scale to the nearest, over the rows of a block (K and V each for itself), once all of them are there
//   read    code * scale, rounded to bf16
// Both move each byte once; HBM bounds them where there are many rows, two dependent loads where there are few.
#include "cache8.cuh"

namespace pk {
namespace {

// A thread block per 64 rows - a block of 64 or several smaller ones - or per block of 128, a warp per row of K and V: 8 values a lane, eight rows a warp.  The values of blocks that are now whole
// stay in registers between the maxima and the codes.  B200, a prompt of 32749 rows of 8 heads (201 MB), us: 38 for blocks of 64, 5.4 TB/s; 42 for blocks of
// 16, 65 with a thread block for each.
template <int BLOCK> struct Append8 {
  static constexpr int warps = BLOCK == 128 ? 16 : 8, rows = BLOCK < 64 ? 64 : BLOCK, blocks = rows / BLOCK, per = rows / warps;
};
template <int BLOCK, bool E4M3>
__global__ void __launch_bounds__(32 * Append8<BLOCK>::warps, BLOCK == 128 ? 2 : 4)
    cache8_append_kernel(const __grid_constant__ Cache8 c, const uint16_t* k, const uint16_t* v, int64_t k_b, int64_t k_t, int64_t k_h, int64_t v_b, int64_t v_t, int64_t v_h,
                         const int32_t* lengths, const int32_t* counts, int T) {
  constexpr int WARPS = Append8<BLOCK>::warps, NB = Append8<BLOCK>::blocks, N = Append8<BLOCK>::per;
  __shared__ uint32_t s_max[NB][WARPS][2];
  pdl_wait();
  pdl_trigger();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, kv = lane >> 4, ch = (lane & 15) * 8;
  const int64_t b = blockIdx.z, h = blockIdx.y;
  const uint16_t* from = kv ? v + b * v_b + h * v_h + ch : k + b * k_b + h * k_h + ch;
  const int64_t from_t = kv ? v_t : k_t;
  const bool few = T <= WARPS;   // a step: a warp per new row, which is asked for together with the lengths
  uint4 fresh = make_uint4(0, 0, 0, 0);
  if (few && blockIdx.x == 0 && warp < T) fresh = *reinterpret_cast<const uint4*>(from + warp * from_t);
  const int n = counts ? min(max(counts[b], 0), T) : T;
  const int64_t len = lengths[b], start = len - n, first = start > 0 ? start : 0, end = len < c.cap ? len : c.cap;
  if (first >= end || n == 0) return;
  const int64_t j0 = first >> c.shift, j = j0 + (int64_t)blockIdx.x * NB, row0 = j << c.shift;   // the first block of this thread block
  if (row0 >= end) return;
  uint16_t* ring = c.recent + b * c.r_b + h * c.r_h + kv * c.r_kv + ch;
  auto place = [&](int64_t r) { return ring + (r % c.R) * c.r_l; };
  const int whole = (int)min((int64_t)NB, (end >> c.shift) - j);   // blocks that are whole now
  auto block_of = [&](int i) { return i * WARPS / BLOCK; };        // of row i of a warp
  if (whole > 0) {
    uint4 x[N];
    const uint16_t* src = from + (row0 + warp - start) * from_t;
#pragma unroll
    for (int i = 0; i < N; i++, src += WARPS * from_t) {
      const int64_t r = row0 + WARPS * i + warp;
      if (block_of(i) < whole) x[i] = *reinterpret_cast<const uint4*>(r >= first ? src : place(r));
      else x[i] = make_uint4(0, 0, 0, 0);
    }
    uint32_t m[NB] = {};
#pragma unroll
    for (int i = 0; i < N; i++) {
      uint32_t& y = m[block_of(i)];
      y = __vimax3_u16x2(y, x[i].x & 0x7fff7fffu, x[i].y & 0x7fff7fffu);
      y = __vimax3_u16x2(y, x[i].z & 0x7fff7fffu, x[i].w & 0x7fff7fffu);
    }
#pragma unroll
    for (int g = 0; g < NB; g++) {
      m[g] = max(m[g] & 0xffffu, m[g] >> 16);
#pragma unroll
      for (int off = 8; off > 0; off >>= 1) m[g] = max(m[g], __shfl_xor_sync(0xffffffffu, m[g], off));
      if ((lane & 15) == 0) s_max[g][warp][kv] = m[g];
    }
    __syncthreads();
    uint8_t* codes = c.codes + b * c.c_b + h * c.c_h + kv * c.c_kv + ch + (row0 + warp) * c.c_l;
#pragma unroll
    for (int g = 0; g < NB; g++) {
      if (g >= whole) break;
      uint32_t top = m[g];
#pragma unroll
      for (int i = 0; i < WARPS; i++) top = max(top, s_max[g][i][kv]);
      const float amax = bf2f((uint16_t)top);
      const bool fine = top < 0x7f80u;
      const Coder16<E4M3> code(amax);
      auto store = [&](auto encode) {
#pragma unroll
        for (int i = g * (N / NB); i < (g + 1) * (N / NB); i++) {
          const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
          float y[8];
#pragma unroll
          for (int e = 0; e < 8; e++) y[e] = __uint_as_float(e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16);
          *reinterpret_cast<uint2*>(codes + WARPS * i * c.c_l) = encode(y);
        }
      };
      if (!fine) store([](const float (&)[8]) { return make_uint2(0, 0); });
      else if (!code.plain) store([&](const float (&y)[8]) { return code.divided(y); });
      else store(code);
      if (warp == 0 && (lane & 15) == 0) c.scales[b * c.s_b + h * c.s_h + (j + g) * c.s_j + kv * c.s_kv] = fine ? __fdiv_rn(amax, CodeScale<E4M3>::MOST) : NAN;
    }
  }
  // The last R rows stay in 16 bits.  Rows of the first block that were there before may lie where new ones go: the thread block that reads them also
  // writes what replaces them.
  const int places = c.R >> c.shift;
  const bool old = first > j0 << c.shift;
  const int64_t kept = max(first, end - c.R);   // the first new row that is kept
  auto keep = [&](int64_t jj) {
    for (int64_t r = max(jj << c.shift, kept) + warp; r < min((jj + 1) << c.shift, end); r += WARPS)
      *reinterpret_cast<uint4*>(place(r)) = *reinterpret_cast<const uint4*>(from + (r - start) * from_t);
  };
  if (few) {   // the first thread block, which alone reads rows that were there, writes all that are new
    if (blockIdx.x != 0) return;
    if (old) __syncthreads();
    if (warp < n && start + warp >= kept && start + warp < end) *reinterpret_cast<uint4*>(place(start + warp)) = fresh;
    return;
  }
  if (row0 + Append8<BLOCK>::rows <= kept && !(old && j == j0)) return;
  if (old && j == j0) __syncthreads();
#pragma unroll 1
  for (int g = 0; g < NB; g++) {
    const int64_t jj = j + g;
    if (!old || (jj - j0) % places != 0) {
      keep(jj);
    } else if (jj == j0) {
      int64_t at = j0;
      if ((kept >> c.shift) > j0) at += ((kept >> c.shift) - j0 + places - 1) / places * places;
      for (; at << c.shift < end; at += places) keep(at);
    }
  }
}

// A warp per row, eight rows in flight; four where they are listed, which are fewer.
template <bool E4M3, bool LISTED>
__global__ void __launch_bounds__(256) cache8_read_kernel(const __grid_constant__ Cache8 c, const int32_t* lengths, const int64_t* rows, uint16_t* out, int64_t o_b, int64_t o_h, int64_t o_l,
                                                          int64_t o_kv, int64_t n) {
  constexpr int N = LISTED ? 4 : 8;
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, kv = lane >> 4, ch = (lane & 15) * 8;
  const int64_t b = blockIdx.z, h = blockIdx.y, i0 = ((int64_t)blockIdx.x * 8 + warp) * N;
  const int64_t len = min((int64_t)max(lengths[b], 0), c.cap), whole = len >> c.shift << c.shift;
  if (i0 >= (LISTED ? n : min(n, len))) return;
  const uint8_t* codes = c.codes + b * c.c_b + h * c.c_h + kv * c.c_kv + ch;
  const float* scales = c.scales + b * c.s_b + h * c.s_h + kv * c.s_kv;
  const uint16_t* ring = c.recent + b * c.r_b + h * c.r_h + kv * c.r_kv + ch;
  uint16_t* to = out + b * o_b + h * o_h + kv * o_kv + ch;
  int64_t r[N];
  uint2 x[N];
  float s[N];
#pragma unroll
  for (int i = 0; i < N; i++) r[i] = LISTED ? (i0 + i < n ? rows[(b * c.H + h) * n + i0 + i] : -1) : i0 + i;
#pragma unroll
  for (int i = 0; i < N; i++) {
    const bool ok = r[i] >= 0 && r[i] < whole;
    x[i] = ok ? *reinterpret_cast<const uint2*>(codes + r[i] * c.c_l) : make_uint2(0, 0);
    s[i] = ok ? scales[(r[i] >> c.shift) * c.s_j] : 0.0f;
  }
#pragma unroll
  for (int i = 0; i < N; i++) {
    uint4 o = make_uint4(0, 0, 0, 0);
    if (r[i] >= whole && r[i] < len) {
      o = *reinterpret_cast<const uint4*>(ring + (r[i] % c.R) * c.r_l);
    } else if (r[i] >= 0 && r[i] < whole) {
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const uint32_t four = e < 2 ? x[i].x : x[i].y;
        float2 f;
        if (E4M3) f = e4m3_floats(four >> (16 * (e & 1)) & 0xffffu);
        else f = make_float2(i8_float(four ^ 0x80808080u, 2 * (e & 1)), i8_float(four ^ 0x80808080u, 2 * (e & 1) + 1));
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[e]) : "f"(__fmul_rn(f.y, s[i])), "f"(__fmul_rn(f.x, s[i])));
      }
      o = make_uint4(w[0], w[1], w[2], w[3]);
    }
    if (LISTED ? i0 + i < n : r[i] < min(n, len)) *reinterpret_cast<uint4*>(to + (i0 + i) * o_l) = o;
  }
}

int lengths_ok(const pk_tensor* lengths, int64_t bs) {
  PK_CHECK_TENSOR(lengths, PK_I32, 1);
  PK_REQUIRE(lengths->shape[0] == bs && is_contig(lengths), "lengths must be contiguous i32 [bs]");
  return PK_OK;
}

}  // namespace
}  // namespace pk

using namespace pk;

extern "C" int pk_cache8_append(const pk_cache8* cache, const pk_tensor* keys, const pk_tensor* values, const pk_tensor* lengths, const pk_tensor* counts, void* stream) {
  Cache8 c = {};
  if (const int rc = fill_cache8(&c, cache, true)) return rc;
  const int64_t bs = cache->codes->shape[0];
  PK_CHECK_TENSOR(keys, PK_BF16, 4);
  PK_CHECK_TENSOR(values, PK_BF16, 4);
  PK_REQUIRE(keys->shape[0] == bs && keys->shape[2] == c.H && keys->shape[3] == 128 && keys->shape[1] < (1LL << 31) - 256, "keys must be bf16 [bs,T,H,128]");
  for (int i = 0; i < 4; i++) PK_REQUIRE(values->shape[i] == keys->shape[i], "values must have the shape of keys");
  PK_REQUIRE(row_tensor(keys) && row_tensor(values), "keys and values need a unit inner stride, other strides that are multiples of 8, and 16-byte alignment");
  if (const int rc = lengths_ok(lengths, bs)) return rc;
  if (counts) {
    PK_CHECK_TENSOR(counts, PK_I32, 1);
    PK_REQUIRE(counts->shape[0] == bs && is_contig(counts), "counts must be contiguous i32 [bs]");
  }
  const int T = (int)keys->shape[1], block = 1 << c.shift;
  if (bs == 0 || T == 0 || c.cap == 0) return PK_OK;
  const int64_t touched = (T + block - 2) / block + 1, per = block < 64 ? 64 / block : 1;
  const dim3 grid((unsigned)((touched + per - 1) / per), (unsigned)c.H, (unsigned)bs);
  const cudaStream_t st = (cudaStream_t)stream;
  StageTimer timer(ST_APPEND, st);
  const bool e4m3 = cache->codes->dtype == PK_E4M3;
#define PK_LAUNCH(B, E)                                                                                                                                                     \
  launch_chain(cache8_append_kernel<B, E>, grid, dim3(32 * Append8<B>::warps), 0, st, c, (const uint16_t*)keys->data, (const uint16_t*)values->data, keys->stride[0], keys->stride[1], keys->stride[2], \
               values->stride[0], values->stride[1], values->stride[2], (const int32_t*)lengths->data, (const int32_t*)(counts ? counts->data : nullptr), T)
#define PK_BLOCK(B) e4m3 ? PK_LAUNCH(B, true) : PK_LAUNCH(B, false)
  block == 16 ? (PK_BLOCK(16)) : block == 32 ? (PK_BLOCK(32)) : block == 64 ? (PK_BLOCK(64)) : (PK_BLOCK(128));
#undef PK_BLOCK
#undef PK_LAUNCH
  return check_launch("cache8_append");
}

extern "C" int pk_cache8_read(const pk_cache8* cache, const pk_tensor* lengths, const pk_tensor* rows, const pk_tensor* out, void* stream) {
  Cache8 c = {};
  if (const int rc = fill_cache8(&c, cache, false)) return rc;
  const int64_t bs = cache->codes->shape[0];
  if (const int rc = lengths_ok(lengths, bs)) return rc;
  PK_CHECK_TENSOR(out, PK_BF16, 5);
  const int64_t n = out->shape[2];
  PK_REQUIRE(out->shape[0] == bs && out->shape[1] == c.H && out->shape[3] == 2 && out->shape[4] == 128 && n < (1LL << 31) - 256, "out must be bf16 [bs,H,n,2,128]");
  PK_REQUIRE(row_tensor(out) && apart(out), "out needs a unit inner stride, other strides that are multiples of 8, 16-byte alignment, and must not share memory within itself");
  if (rows) {
    PK_CHECK_TENSOR(rows, PK_I64, 3);
    PK_REQUIRE(rows->shape[0] == bs && rows->shape[1] == c.H && rows->shape[2] == n && is_contig(rows), "rows must be contiguous i64 [bs,H,n], n as in out");
  } else {
    PK_REQUIRE(n <= c.cap, "out has more rows than the cache");
  }
  if (bs == 0 || n == 0) return PK_OK;
  const int per = rows ? 32 : 64;
  const dim3 grid((unsigned)((n + per - 1) / per), (unsigned)c.H, (unsigned)bs);
  const cudaStream_t st = (cudaStream_t)stream;
  StageTimer timer(ST_GATHER, st);
#define PK_LAUNCH(E, L)                                                                                                                                                           \
  launch_chain(cache8_read_kernel<E, L>, grid, dim3(256), 0, st, c, (const int32_t*)lengths->data, (const int64_t*)(rows ? rows->data : nullptr), (uint16_t*)out->data, out->stride[0], \
               out->stride[1], out->stride[2], out->stride[3], n)
  if (cache->codes->dtype == PK_E4M3) rows ? PK_LAUNCH(true, true) : PK_LAUNCH(true, false);
  else rows ? PK_LAUNCH(false, true) : PK_LAUNCH(false, false);
#undef PK_LAUNCH
  return check_launch("cache8_read");
}
