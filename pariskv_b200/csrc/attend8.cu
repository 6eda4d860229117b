// Attention of the last tokens of the sequences over the cache in 8 bits:  o = sum_j p_j v_j / sum_j p_j,  p_j = 2^((s_j - max s) scale log2 e),
//   s_j = ks (q . kc_j),  p_j v_j = (p_j vs) vc_j    with codes kc, vc of a row and the scales ks, vs of its block.
//
// HBM bounds a step: 256 bytes a row.  The products run on mma.sync, whose operands of 16 bits hold codes and queries exactly: keys and queries as fp16, which takes the fewest instructions, the queries after a power of
// two per row, or as bf16 where a query's values are too far apart for that (and always from 17 query rows on).  A weight times the scale of the values is taken as two bf16 numbers, 17 bits whatever its size, and the
// values' codes as bf16: one fp16 number for it, under a power of two per query row that follows the largest, has 11 bits down to 2^-14 of the largest and none below 2^-25, so that a long tail behind one key of most of
// the weight and a value near zero is lost.  (B200, us, one fp16 | two bf16: 128K keys 53.4 | 53.7, 16 sequences of 16 - 32K 136 | 136, after a second of them 138 | 141, 32 query rows over 8 x 58K 44.5 | 52.5.)
// tcgen05, with rows of the cache as the 128 rows of an operand, would want the codes in 16 bits in shared memory first.
// The rows behind the last whole block come from `recent` as bf16, their weights as two bf16 numbers each too.
//
// Every warp is by itself: 32 rows a step from global memory into its own stages of shared memory by cp.async, one step ahead, at any strides.  The order of channels in Q K^T and of rows in P V is free, and
// chosen so that a lane's fragments of K are 32 consecutive codes of a row, and those of V 16 consecutive codes of four rows.
// Tiles of 128 rows, four warps of a block side by side.  Short caches: a cluster of blocks per item (sample, KV head, group of query rows), one launch.  Others: the tiles of all items, laid end to end, are cut
// into equal ranges as in attend_few.cu, and attend8_merge_kernel joins the records of items that are cut.
//
// B200, us, replayed graphs.  128K keys of 8 heads, a token of four queries each (269 MB) 53.7: blocks begin their rows 2 us after the start and end after 33 to 49, as fast as their SMs get them (with the products left
// out the whole takes 46), the joining launch takes 2; 16 sequences of 16 - 32K (e4m3) 136, 6.0 TB/s; 32 query rows a KV head over 8 x 58K keys 52: eight warps an SM by their registers, tensor cores busy 46 % of the
// time, the rest they wait for one another's turn.
// Steps of the form with one fp16 number for a weight: loops by segment with one scaling for the 16 rows that share a scale, 100 -> 60; less code around the loops (run once, it costs its fetching) 97 -> 60 for 32 rows; query rows across and a lazy maximum
// 56 -> 55, 60 -> 52; ranges that end where the items do 50 -> 47; queries asked for before the rows, two steps of copies at once, all records under way 47.6 -> 44.5.  No better: three stages, two blocks an SM
// (52 - 54), two ranges a place (58; of long ranges they are kept), two scores an instruction.
#include <type_traits>

#include "cache8.cuh"
#include "tiles.cuh"

namespace pk {
namespace {

constexpr int A8_TILE = 128, A8_THREADS = 128;
constexpr int A8_STAGE = 8192;                    // 32 rows of K and V in codes, 16 in bf16
constexpr int A8_SLOT = A8_STAGE + 16;            // and the scales: K of the first and second 16 rows, V of them
constexpr int A8_QS = 272;                        // bytes between two rows of the queries in bf16
// ROWS: query rows of an item.
template <int ROWS> struct A8 {
  static constexpr bool across = ROWS == 8;       // query rows are the columns of the products, rows of the cache and channels their rows: eight fill an operand
  static constexpr int ctas = ROWS == 32 ? 2 : 3, q_bytes = ROWS * (256 + A8_QS), smem = 4 * 2 * A8_SLOT + q_bytes;
  // A warp's partial of eight rows, in floats: channels lie in runs of `run`, padded so that the stores fall into all banks.
  static constexpr int run = across ? 16 : 32, step = across ? 164 : 144;
  static __device__ __forceinline__ int place(int row, int channel) { return row * step + channel / run * (run + 4) + channel % run; }
  static_assert(8 * step * 4 <= A8_STAGE, "the partial takes the place of a stage");
};

struct Attend8 {
  Cache8 c;
  const uint16_t* q;
  int64_t q_b, q_t, q_h;
  const int32_t* lengths;
  int bs, T, G, row_groups, cluster;   // cluster: blocks that share an item, 0 where the ranges do not follow the items
  float scale_log2;
  uint16_t* out;
  float *lse, *records;   // records: [2 * blocks][ROWS * 130]
};

__device__ __forceinline__ int len8(const Attend8& p, int b) { return (int)min((int64_t)max(p.lengths[b], 0), p.c.cap); }
__device__ __forceinline__ int tiles8(const Attend8& p, int len) {   // of an item: whole blocks, then the rows behind them
  const int whole = len >> p.c.shift << p.c.shift;
  return max(1, (whole + A8_TILE - 1) / A8_TILE + (whole < len));
}

// Where every item has eight blocks' tiles or more, the ranges end where the items do: the blocks whose range would begin in an item share it evenly.  A range over the end of an item costs its block
// another set of queries and another sum over its warps, 4 us that the whole launch waits for.  first8: the first of an item's blocks, `at` its first tile.
__device__ __forceinline__ bool apart8(int64_t total, int fewest, unsigned shares) { return (int64_t)fewest * shares >= 8 * total; }
__device__ __forceinline__ unsigned first8(int64_t at, int64_t total, unsigned shares) {
  return total < 1 << 22 ? ((unsigned)at * shares + (unsigned)total - 1) / (unsigned)total : (unsigned)((at * shares + total - 1) / total);
}
// The fewest tiles of an item, by a warp.
__device__ __forceinline__ int fewest8(const Attend8& p) {
  int n = 0x7fffffff;
  for (int b = threadIdx.x & 31; b < p.bs; b += 32) n = min(n, tiles8(p, len8(p, b)));
  return __reduce_min_sync(0xffffffffu, n);
}
// By a warp: the tiles of all items (below 2^31: the launch sees to it), the fewest of one, and the sample with the tile that the block's range begins with.
struct Plan8 {
  unsigned total, before, begin;   // before: tiles of the samples before `sample`; begin: of the range
  int sample, fewest;
};
__device__ __forceinline__ Plan8 plan8(const Attend8& p, unsigned items, unsigned block, unsigned blocks) {
  const int lane = threadIdx.x & 31;
  Plan8 r = {0, 0, 0, 0, 0x7fffffff};
  unsigned first = 0;
  for (int b0 = 0; b0 < p.bs; b0 += 32) {
    const int n = b0 + lane < p.bs ? tiles8(p, len8(p, b0 + lane)) : 0;
    if (b0 == 0) first = n * items;
    r.total += __reduce_add_sync(0xffffffffu, n * items), r.fewest = min(r.fewest, n == 0 ? 0x7fffffff : n);
  }
  r.fewest = __reduce_min_sync(0xffffffffu, r.fewest);
  const unsigned at = r.begin = (unsigned)share_begin(r.total, block, min(blocks, r.total));
  for (int b0 = 0; b0 < p.bs; b0 += 32) {
    const unsigned mine = b0 == 0 ? first : b0 + lane < p.bs ? items * tiles8(p, len8(p, b0 + lane)) : 0;
    unsigned end = mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const unsigned o = __shfl_up_sync(0xffffffffu, end, off);
      if (lane >= off) end += o;
    }
    const unsigned past = __ballot_sync(0xffffffffu, b0 + lane < p.bs && r.before + end > at);
    if (past) {
      const int i = __ffs(past) - 1;
      r.sample = b0 + i, r.before += __shfl_sync(0xffffffffu, end - mine, i);
      return r;
    }
    r.before += __shfl_sync(0xffffffffu, end, 31);
  }
  return r;
}

// A block's way through its range: segments of consecutive tiles of one item.
struct Way8 {
  int b, h, group, len, whole, n, tile;
  int64_t left;   // tiles of the range that are left
  __device__ __forceinline__ void sample(const Attend8& p) { len = len8(p, b), whole = len >> p.c.shift << p.c.shift, n = tiles8(p, len); }
  __device__ __forceinline__ int count() const { return (int)min((int64_t)(n - tile), left); }
  __device__ __forceinline__ void next(const Attend8& p) {
    left -= count();
    tile = 0;
    if (++group < p.row_groups) return;
    group = 0;
    if (++h < p.c.H) return;
    h = 0;
    if (++b < p.bs) sample(p);
  }
};

__device__ __forceinline__ void cp16(unsigned dst, const void* src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ void cp16(unsigned dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp4(unsigned dst, const void* src) { asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
  __syncwarp();
}
// Reads that the compiler may move between the barriers: plain loads of the block's shared memory, at an offset.
extern __shared__ __align__(128) unsigned char dyn8[];
__device__ __forceinline__ uint4 lds16(unsigned off) { return *reinterpret_cast<const uint4*>(dyn8 + off); }
__device__ __forceinline__ uint2 lds8(unsigned off) { return *reinterpret_cast<const uint2*>(dyn8 + off); }
__device__ __forceinline__ uint32_t half2_of(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ void mma_f16(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Two codes as bf16 numbers.  Whole numbers, the last bytes of the halves of w: 128 + the last seven bits, and 128, or 256 where the code is below zero, is taken off.  (As lop3 by hand: the compiler's own form of the two
// masks, with constants on both sides, takes twice the instructions, 128K keys 65 us for 54.)
__device__ __forceinline__ uint32_t i8_pair(uint32_t w) {
  uint32_t r;
  asm("{\n\t.reg .b32 x, y;\n\tlop3.b32 x, %1, 0x007f007f, 0x43004300, 0xea;\n\tlop3.b32 y, %1, 0x00800080, 0x43004300, 0xea;\n\tsub.rn.bf16x2 %0, x, y;\n\t}" : "=r"(r) : "r"(w));
  return r;
}
// e4m3, each continued by its sign to 16 bits: its seven bits as the last of the exponent and the first of the fraction, 2^-120 of the number (below 2^-126: a bf16 number without a leading one, exactly)
__device__ __forceinline__ uint32_t e4m3_pair(uint32_t w) { return w << 4 & 0x87f087f0u; }
template <int SELECT>
__device__ __forceinline__ uint32_t bytes_of(uint32_t a, uint32_t b) {   // with the sign's form of a selector
  uint32_t r;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "n"(SELECT));
  return r;
}
// K: two codes of w as fp16 numbers, which takes less than as bf16.  Whole numbers: codes 0 and 2 (hi: 1 and 3) become the last bits of 1024 + (code + 128), and 1152 is taken off.  e4m3: codes 0 and 1 (hi: 2
// and 3).  WIDE: as bf16 numbers, codes 0 and 2 (hi: 1 and 3), of e4m3 2^-120 of them.  The queries lie in the same order.
template <bool E4M3, bool WIDE>
__device__ __forceinline__ uint32_t codes_lo(uint32_t w) {
  if (WIDE) return E4M3 ? e4m3_pair(bytes_of<0xa280>(w, w)) : i8_pair(w);
  uint32_t r;
  if (E4M3) asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\t}" : "=r"(r) : "r"(w));
  else asm("{\n\t.reg .b32 x;\n\tlop3.b32 x, %1, 0x00ff00ff, 0x64806480, 0x6a;\n\tadd.rn.f16x2 %0, x, %2;\n\t}" : "=r"(r) : "r"(w), "r"(0xe480e480u));
  return r;
}
template <bool E4M3, bool WIDE>
__device__ __forceinline__ uint32_t codes_hi(uint32_t w) {
  if (WIDE) return E4M3 ? e4m3_pair(bytes_of<0xb391>(w, w)) : i8_pair(w >> 8);
  uint32_t r;
  if (E4M3) asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, b;\n\t}" : "=r"(r) : "r"(w));
  else r = codes_lo<false, false>(w >> 8);
  return r;
}
// V: code I of words a and c, which are of two rows
template <bool E4M3, int I>
__device__ __forceinline__ uint32_t codes_of(uint32_t a, uint32_t c) {
  if (!E4M3) return i8_pair(bytes_of<(4 + I) << 8 | I>(a, c));
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(e4m3_pair(bytes_of<(12 + I) << 12 | (4 + I) << 8 | (8 + I) << 4 | I>(a, c))), "r"(0x7b807b80u));
  return r;
}
// Weights as two bf16 numbers each, 17 bits: pairs of them, and of what their rounding leaves
__device__ __forceinline__ void two_of(float a, float c, uint32_t& hi, uint32_t& lo) {
  hi = pack2(a, c), lo = pack2(a - __uint_as_float(hi << 16), c - __uint_as_float(hi & 0xffff0000u));
}
// (a, b) (c, d) + (e, f), and (a, b) (c, d): two fp32 operations in one instruction
__device__ __forceinline__ float2 fma2(float a, float b, float c, float d, float e, float f) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\tfma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a), "f"(b), "f"(c), "f"(d), "f"(e), "f"(f));
  return r;
}
__device__ __forceinline__ float2 mul2(float a, float b, float c, float d) {
  float2 r;
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}" : "=f"(r.x), "=f"(r.y) : "f"(a), "f"(b), "f"(c), "f"(d));
  return r;
}
// Rows and columns of 8 x 8 numbers of 16 bits change places.
__device__ __forceinline__ uint32_t turn(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}

// Running state of one of a lane's query rows.  m: the largest score when it was last looked for, times log2 e / sqrt d; l: the sum of p over this lane's scores, relative to 2^m, as O is.
struct RowState {
  float m, l;
};
// To a new largest score: what O has to be multiplied by.
__device__ __forceinline__ float move(RowState& s, float m) {
  const float f = s.m == -INFINITY ? 0.0f : m > s.m ? ex2(s.m - m) : 1.0f;
  s.m = m, s.l *= f;
  return f;
}
// The same place in the shared memory of block `rank` of the cluster.
__device__ __forceinline__ float remote(const void* at, int rank) {
  float r;
  asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %1, %2;\n\tld.shared::cluster.f32 %0, [a];\n\t}" : "=f"(r) : "r"(smem_addr(at)), "r"(rank) : "memory");
  return r;
}
__device__ __forceinline__ float4 remote4(const void* at, int rank) {
  float4 r;
  asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %4, %5;\n\tld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [a];\n\t}" : "=f"(r.x), "=f"(r.y), "=f"(r.z), "=f"(r.w) : "r"(smem_addr(at)), "r"(rank) : "memory");
  return r;
}
__device__ __forceinline__ void cluster_sync() { asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// PAIRED: up to four query rows.  They are columns 0 to 3 of the products and 4 to 7 too, and the second parts of the weights are the weights of the latter, so that one product has both
// (16 sequences of 16 - 32K, after a second of them, e4m3 146 -> 143 us, int8 157 -> 152).
template <bool E4M3, int ROWS, bool DENSE, bool PAIRED>
__global__ void __launch_bounds__(A8_THREADS, A8<ROWS>::ctas) attend8_kernel(const __grid_constant__ Attend8 p) {
  constexpr bool ACROSS = A8<ROWS>::across;
  constexpr int MT = ROWS == 32 ? 2 : 1, NR = 2 * MT;   // operands of 16 query rows; query rows that a lane's scores belong to: 8 e + g, across 2 t4 + e
  constexpr int NV = ACROSS ? 4 : 8;                    // its scores of each in a step
  constexpr bool NARROW = ROWS < 32;                    // queries and keys' codes as fp16 where that is exact (of 32 rows the two forms do not fit into the registers)
  __shared__ float s_m[4][ROWS], s_l[4][ROWS], s_factor[ROWS], s_M[ROWS], s_L[ROWS];   // of the warps; of the block, for its cluster
  __shared__ Way8 s_way;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  pdl_wait();
  pdl_trigger();
  const int blocks = (int)gridDim.x;
  const int64_t items = (int64_t)p.c.H * p.row_groups;
  const int n_rows_all = p.T * p.G, Hq = p.c.H * p.G;
  // 16 channels of query row `row` of an item for this thread, eight of them a row
  auto query = [&](int b, int h, int group, int row, uint4 (&x)[2]) {
    const int r = group * ROWS + min(PAIRED ? row & 3 : row, min(ROWS, n_rows_all - group * ROWS) - 1);
    const uint4* from = reinterpret_cast<const uint4*>(p.q + b * p.q_b + (int64_t)(r / p.G) * p.q_t + (int64_t)(h * p.G + r % p.G) * p.q_h + 16 * (tid & 7));
    x[0] = from[0], x[1] = from[1];
  };
  Way8 way;
  uint4 q_first[2];   // a cluster knows its item before it knows the lengths: its queries come together with them
  if (p.cluster) {
    const int item = (int)blockIdx.x / p.cluster, rank = (int)blockIdx.x % p.cluster;
    way.b = item / (int)items, way.h = item % (int)items / p.row_groups, way.group = item % p.row_groups;
    if (ROWS <= 16) query(way.b, way.h, way.group, tid >> 3, q_first);
    way.sample(p);
    way.tile = way.n * rank / p.cluster, way.left = way.n * (rank + 1) / p.cluster - way.tile;
    if (tid < ROWS) s_M[tid] = -INFINITY, s_L[tid] = 0.0f;
  } else {
    if (warp == 0) {   // (a division of whole numbers is some forty instructions: two lanes do two of a kind at once)
      const Plan8 plan = plan8(p, (unsigned)items, blockIdx.x, (unsigned)blocks);
      const unsigned shares = min((unsigned)blocks, plan.total);
      Way8 w = {};
      w.b = plan.sample;
      if (blockIdx.x < shares) {
        w.sample(p);
        const unsigned n = (unsigned)w.n, at = plan.begin - plan.before, item = at / n;
        w.h = (int)item, w.group = 0;
        if (p.row_groups > 1) w.h = (int)(item / (unsigned)p.row_groups), w.group = (int)(item % (unsigned)p.row_groups);
        if (apart8(plan.total, plan.fewest, shares)) {
          const unsigned c = first8(plan.before + (item + (lane & 1)) * n, plan.total, shares), c0 = __shfl_sync(0xffffffffu, c, 0), cnt = __shfl_sync(0xffffffffu, c, 1) - c0;
          const unsigned t = (unsigned)share_begin(n, blockIdx.x - c0 + (lane & 1), cnt);
          w.tile = (int)__shfl_sync(0xffffffffu, t, 0), w.left = __shfl_sync(0xffffffffu, t, 1) - (unsigned)w.tile;
        } else {
          w.tile = (int)(at - item * n), w.left = share_begin(plan.total, blockIdx.x + 1, shares) - plan.begin;
        }
      }
      if (lane == 0) s_way = w;
    }
    __syncthreads();
    way = s_way;
    if (way.left == 0) return;
  }
  const unsigned base = smem_addr(dyn8), mine = A8<ROWS>::q_bytes + warp * 2 * A8_SLOT, q_off = (ROWS == 8 ? 8 : 16) * lane;   // offsets in the block's shared memory
  for (; way.left > 0; way.next(p)) {
    // ---- a segment ----
    const int b = way.b, h = way.h, group = way.group, whole = way.whole, count = way.count();
    const bool whole_item = count == way.n && p.cluster <= 1;
    const int coded = (whole + A8_TILE - 1) / A8_TILE;                          // tiles of codes of the item
    const int n_coded = max(0, min(coded, way.tile + count) - way.tile);        // of the segment
    const bool recent = way.len > whole && way.tile + count == way.n;
    const int n_rows = min(ROWS, n_rows_all - group * ROWS);
    int row0 = way.tile * A8_TILE + 32 * warp;
    // A step's 32 rows on their way.  A chunk of 16 bytes lies where its row's number moves it, so that the reads below fall into all banks.
    const int ck = lane & 7, ckv = lane >> 3 & 1, odd = lane >> 4;
    const uint8_t* src = p.c.codes + b * p.c.c_b + h * p.c.c_h + ckv * p.c.c_kv + (int64_t)(row0 + odd) * p.c.c_l + ck * 16;
    const float* scales = p.c.scales + b * p.c.s_b + h * p.c.s_h + (lane >> 1 & 1) * p.c.s_kv;
    auto load = [&](int slot) {
      const unsigned to = base + mine + slot * A8_SLOT, chunk = to + ckv * 4096 + odd * 128;
      const int live = whole - row0;
      const int64_t c_l = DENSE ? 256 : p.c.c_l;
      if (live >= 32) {
        const uint8_t* from = src;
#pragma unroll
        for (int i = 0; i < 16; i++, from += 2 * c_l) cp16(chunk + i * 256 + ((ck ^ (ckv ? (2 * i) & 6 : odd)) << 4), from);
      } else if (live > 0) {
#pragma unroll
        for (int i = 0; i < 16; i++) cp16(chunk + i * 256 + ((ck ^ (ckv ? (2 * i) & 6 : odd)) << 4), 2 * i + odd < live ? src + 2 * i * c_l : src - odd * c_l, 2 * i + odd < live);
      }
      if (lane < 4 && live > 0) cp4(to + A8_STAGE + 4 * lane, scales + (int64_t)(min(row0 + 16 * (lane & 1), whole - 1) >> p.c.shift) * p.c.s_j);
      cp_commit();
      src += A8_TILE * c_l, row0 += A8_TILE;
    };
    auto load_recent = [&](int sub, int slot) {   // 16 rows in 16 bits: those of the four warps follow one another, so that blocks of up to 64 rows need one turn
      const int r0 = whole + 64 * sub + 16 * warp, live = min(16, way.len - r0), kv = lane >> 4;
      const uint16_t* ring = p.c.recent + b * p.c.r_b + h * p.c.r_h + kv * p.c.r_kv + (lane & 15) * 8;
      const unsigned to = base + mine + slot * A8_SLOT + kv * 4096 + (lane & 15) * 16;
      if (live > 0) {
        int place = r0 % p.c.R;
#pragma unroll 4
        for (int i = 0; i < 16; i++, place = place + 1 == p.c.R ? 0 : place + 1) cp16(to + i * 256, ring + (int64_t)(i < live ? place : r0 % p.c.R) * p.c.r_l, i < live);
      }
      cp_commit();
    };
    // Steps of the segment: its tiles of codes, then two of rows in 16 bits.  A group of copies for each, without any where there is none.
    auto load_step = [&](int j) {
      if (j < n_coded) load(j & 1);
      else if (recent && j < n_coded + 2) load_recent(j - n_coded, j & 1);
      else cp_commit();
    };
    // The queries are asked for before the rows, which all blocks ask for at once: behind them they came 2 us later.
    uint4 q_rows[ROWS / 16 + (ROWS == 8)][2];
#pragma unroll
    for (int i = 0; i < (ROWS + 15) / 16; i++) {
      if (ROWS <= 16 && p.cluster) q_rows[i][0] = q_first[0], q_rows[i][1] = q_first[1];
      else query(b, h, group, 16 * i + (tid >> 3), q_rows[i]);
    }
    load_step(0);
    load_step(1);
    // queries: as they are, and as fp16 after a power of two per row in the order in which a lane needs them as operands; eight threads a row.  The largest of a row becomes a number from 2^12 to 2^13 (at the ends
    // of the range less, or up to 2^15), so that all that is not below 2^-29 of it is an fp16 number exactly.  Where a value is, which no model's queries have unless a channel is out of all proportion, the block's
    // queries and its keys' codes become bf16.
    auto stage = [&](auto wide) {
      constexpr bool WIDE = decltype(wide)::value;
      bool far_below = false;
#pragma unroll
      for (int i16 = 0; i16 < (ROWS + 15) / 16; i16++) {
        const int row = 16 * i16 + (tid >> 3), c = tid & 7;   // 16 channels from 16 c on
        const uint4 (&x)[2] = q_rows[i16];
        const uint32_t xw[8] = {x[0].x, x[0].y, x[0].z, x[0].w, x[1].x, x[1].y, x[1].z, x[1].w};
        uint32_t top = 0, low = 0x7fff7fffu;   // low: the smallest that is not zero
#pragma unroll
        for (int i = 0; i < 8; i++) top = __vmaxu2(top, xw[i] & 0x7fff7fffu), low = __vminu2(low, __vsub2(xw[i] & 0x7fff7fffu, 0x00010001u));
        top = max(top & 0xffffu, top >> 16), low = min(low & 0xffffu, low >> 16) + 1;
#pragma unroll
        for (int off = 1; off < 8; off <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, off));
        // a row with an infinity or NaN becomes NaN
        const unsigned ex = max(min(top >> 7, 252u), 16u);
        const bool fine = top < 0x7f80u;
        const float up = fine ? __uint_as_float((254u - ex) << 23) : NAN;
        far_below |= fine && ex > max(low >> 7, 1u) + 29;
        if (row < ROWS) {
          if (c == 0) s_factor[row] = fine ? __uint_as_float((WIDE ? ex : ex - 12) << 23) * p.scale_log2 : NAN;
          if (!WIDE || !NARROW) {
            uint4* raw = reinterpret_cast<uint4*>(dyn8 + ROWS * 256 + row * A8_QS + 32 * c);
            raw[0] = x[0], raw[1] = x[1];
          }
#pragma unroll
          for (int k = 0; k < 4; k++) {
            float f[4] = {__uint_as_float(xw[2 * k] << 16) * up, __uint_as_float(xw[2 * k] & 0xffff0000u) * up, __uint_as_float(xw[2 * k + 1] << 16) * up,
                          __uint_as_float(xw[2 * k + 1] & 0xffff0000u) * up};
#pragma unroll
            for (int i = 0; i < 4; i++) f[i] *= !WIDE ? 0x1p12f : E4M3 ? 0x1p120f : 1.0f;
            const uint32_t lo = WIDE ? pack2(f[0], f[2]) : half2_of(f[0], f[E4M3 ? 1 : 2]), hi = WIDE ? pack2(f[1], f[3]) : half2_of(f[E4M3 ? 2 : 1], f[3]);
            const int s = 4 * (c & 1) + k, of = 4 * (row & 7) + (c >> 1);   // the lane that it is for
            if (ROWS == 8) {
              *reinterpret_cast<uint2*>(dyn8 + s * 256 + of * 8) = make_uint2(lo, hi);
            } else {   // a0, a1 rows g and g + 8 of the first pair of channels, a2, a3 of the second
              uint32_t* to = reinterpret_cast<uint32_t*>(dyn8 + ((row >> 4) * 8 + s) * 512 + of * 16) + (row >> 3 & 1);
              to[0] = lo, to[2] = hi;
            }
          }
        }
      }
      return far_below;
    };
    bool wide = true;
    if constexpr (NARROW) wide = __syncthreads_or(stage(std::false_type()));
    if (wide) {
      stage(std::true_type());
      __syncthreads();
    }
    // O: operand rows g, g + 8 are query rows, the two columns channels 32 t4 + n and + 16; across: the two columns query rows, operand rows channels 16 g + 2 n, + 1
    constexpr int ON = ACROSS ? 8 : 16;
    float o[MT][ON][4] = {};
    RowState st[NR];
    float factor[NR];   // log2 e / sqrt d, and what the row was scaled by
    int last[NR];       // the last row that a query row sees
    const int end = (p.lengths[b] > p.c.cap ? (int)p.c.cap : p.lengths[b]) - p.T;
    auto row_of = [&](int e) { return ACROSS ? 2 * t4 + e : 8 * e + g; };
#pragma unroll
    for (int e = 0; e < NR; e++) {
      st[e] = {-INFINITY, 0.0f};
      factor[e] = s_factor[row_of(e)];
      last[e] = end + (group * ROWS + min(PAIRED ? row_of(e) & 3 : row_of(e), n_rows - 1)) / p.G;
    }
    auto scale_row = [&](int e, float f) {
#pragma unroll
      for (int n = 0; n < ON; n++) {
        if (ACROSS) o[0][n][e & 1] *= f, o[0][n][2 + (e & 1)] *= f;
        else o[e >> 1][n][2 * (e & 1)] *= f, o[e >> 1][n][2 * (e & 1) + 1] *= f;
      }
    };
    auto row_max = [&](float x) {   // over the lanes that have scores of the same query rows
      if (ACROSS) {
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
        return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
      }
      x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
      return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
    };
    const int lim = min(end + group * ROWS / p.G, whole - 1) - 31;   // 32 rows that begin up to here are seen by all
    unsigned at = mine;
    auto coded_rows = [&](auto wide) {
      constexpr bool WIDE = decltype(wide)::value;
      for (int j = 0; j < n_coded; j++) {
        const int first = (way.tile + j) * A8_TILE + 32 * warp;
        at = mine + (j & 1) * A8_SLOT;
        cp_wait<1>();
        if (first >= whole) {
          load_step(j + 2);
          continue;
        }
        // scores of a lane: s[half of the rows][..]: row 8 i + 2 t4 + k of the half (i = c / 4, k = c & 1) and query row g, 8 + g (c >> 1 & 1); across: row g, 8 + g (c >> 1) and query row c & 1
        float s[MT][2][ACROSS ? 4 : 8];
        auto product = [](float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
          if (WIDE) mma_bf16(c, a0, a1, a2, a3, b0, b1);
          else mma_f16(c, a0, a1, a2, a3, b0, b1);
        };
#pragma unroll
        for (int half = 0; half < 2; half++) {
          uint4 kw[2][2];
#pragma unroll
          for (int i = 0; i < 2; i++) {
            const unsigned from = at + (8 * (2 * half + i) + g) * 128;
            kw[i][0] = lds16(from + (((2 * t4) ^ (g & 1)) << 4)), kw[i][1] = lds16(from + (((2 * t4 + 1) ^ (g & 1)) << 4));
          }
#pragma unroll
          for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int c = 0; c < (ACROSS ? 4 : 8); c++) s[mt][half][c] = 0.0f;
#pragma unroll
          for (int ks = 0; ks < 8; ks++) {
            uint32_t b[2][2];
#pragma unroll
            for (int i = 0; i < 2; i++) {
              const uint4 v = kw[i][ks >> 2];
              const uint32_t w = (ks & 3) == 0 ? v.x : (ks & 3) == 1 ? v.y : (ks & 3) == 2 ? v.z : v.w;
              b[i][0] = codes_lo<E4M3, WIDE>(w), b[i][1] = codes_hi<E4M3, WIDE>(w);
            }
            if (ACROSS) {
              const uint2 q = lds8(q_off + ks * 256);
              product(s[0][half], b[0][0], b[1][0], b[0][1], b[1][1], q.x, q.y);
            } else {
#pragma unroll
              for (int mt = 0; mt < MT; mt++) {
                const uint4 q = lds16(q_off + (mt * 8 + ks) * 512);
                product(s[mt][half], q.x, q.y, q.z, q.w, b[0][0], b[0][1]);
                product(s[mt][half] + (ACROSS ? 0 : 4), q.x, q.y, q.z, q.w, b[1][0], b[1][1]);
              }
            }
          }
        }
        float4 sc;   // scales: K of the first and second 16 rows, V of them
        {
          const uint4 x = lds16(at + A8_STAGE);
          sc = make_float4(__uint_as_float(x.x), __uint_as_float(x.y), __uint_as_float(x.z), __uint_as_float(x.w));
        }
        // score v of query row e: half v / (NV / 2), and its row in the step
        auto score = [&](int e, int v) -> float& {
          if (ACROSS) return s[0][v >> 1][2 * (v & 1) + (e & 1)];
          return s[e >> 1][v >> 2][4 * (v >> 1 & 1) + 2 * (e & 1) + (v & 1)];
        };
        auto row_at = [&](int v) { return ACROSS ? 16 * (v >> 1) + 8 * (v & 1) + g : 16 * (v >> 2) + 8 * (v >> 1 & 1) + 2 * t4 + (v & 1); };
        uint32_t pw[NR][NV / 2], pl[NR][NV / 2];   // weights as pairs of bf16 numbers, of the columns 2 t4, 2 t4 + 1, and what their rounding left; across: see below
        float w[NR][NV];
        const bool all = first <= lim;
        bool far = !all;
        // Two scores at a time: neighbours of a query row; across, the two query rows of a row of the cache.
#pragma unroll
        for (int e = 0; e < NR; e += ACROSS ? 2 : 1) {
          const float k0[2] = {sc.x * factor[e], sc.y * factor[e]}, k1[2] = {ACROSS ? sc.x * factor[e + ACROSS] : k0[0], ACROSS ? sc.y * factor[e + ACROSS] : k0[1]};
          const float m0 = -st[e].m, m1 = ACROSS ? -st[e + ACROSS].m : m0;
          float top = -INFINITY;
#pragma unroll
          for (int v = 0; v < NV; v += ACROSS ? 1 : 2) {
            const int h2 = v / (NV / 2);
            const float2 x = ACROSS ? fma2(score(e, v), score(e + ACROSS, v), k0[h2], k1[h2], m0, m1) : fma2(score(e, v), score(e, v + 1), k0[h2], k0[h2], m0, m0);
            top = max3(top, x.x, x.y);
            w[e][v] = x.x;
            if (ACROSS) w[e + ACROSS][v] = x.y;
            else w[e][v + 1] = x.y;
          }
          far |= top > 8.0f;   // the running maximum may lie 2^8 below the true one: then nothing has to be moved
        }
        if (!__any_sync(0xffffffffu, far)) {
#pragma unroll
          for (int e = 0; e < NR; e += ACROSS ? 2 : 1) {
            float sum0 = 0.0f, sum1 = 0.0f;
#pragma unroll
            for (int v = 0; v < NV; v += ACROSS ? 1 : 2) {
              const float z = v / (NV / 2) ? sc.w : sc.z;
              float& a = w[e][v];
              float& c = ACROSS ? w[e + ACROSS][v] : w[e][(v + 1) % NV];
              a = ex2(a), c = ex2(c);
              add2(sum0, sum1, a, c);
              const float2 x = mul2(a, c, z, z);
              a = x.x, c = x.y;
            }
            if (ACROSS) st[e].l += sum0, st[e + ACROSS].l += sum1;
            else st[e].l += sum0 + sum1;
          }
        } else {
#pragma unroll
          for (int e = 0; e < NR; e++) {
            const float kf[2] = {sc.x * factor[e], sc.y * factor[e]}, vs[2] = {sc.z, sc.w};
            float m = st[e].m, sum = 0.0f;
            bool seen[NV];
#pragma unroll
            for (int v = 0; v < NV; v++) {
              seen[v] = all || (first + row_at(v) < whole && first + row_at(v) <= last[e]);
              if (seen[v]) m = fmaxf(m, score(e, v) * kf[v / (NV / 2)]);
            }
            m = row_max(m);
            const float least = m == -INFINITY ? 0.0f : m;
#pragma unroll
            for (int v = 0; v < NV; v++) {
              const float y = seen[v] ? ex2(fmaf(score(e, v), kf[v / (NV / 2)], -least)) : 0.0f;
              sum += y;
              w[e][v] = seen[v] ? y * vs[v / (NV / 2)] : 0.0f;   // (the scale of a block that it does not see may be NaN)
            }
            const float f = move(st[e], m);
            st[e].l += sum;
            if (__any_sync(0xffffffffu, f != 1.0f)) scale_row(e, f);
          }
        }
        // across: pairs are two query rows of one row of the cache; an exchange of 8 x 8 numbers makes them two rows of one query row
        if (ACROSS) {
#pragma unroll
          for (int v = 0; v < 4; v++) {
            uint32_t hi, lo;
            two_of(w[0][v], w[1][v], hi, lo);
            if (PAIRED) {
              pw[v >> 1][v & 1] = turn(t4 < 2 ? hi : lo);
            } else {
              pw[v >> 1][v & 1] = turn(hi), pl[v >> 1][v & 1] = turn(lo);
            }
          }
        } else {
#pragma unroll
          for (int e = 0; e < NR; e++)
#pragma unroll
            for (int v = 0; v < NV; v += 2) two_of(w[e][v], w[e][v + 1], pw[e][v >> 1], pl[e][v >> 1]);
        }
#pragma unroll
        for (int half = 0; half < 2; half++) {
          uint4 v[4];   // rows 2 t4, 2 t4 + 1, and eight further; channels 16 g ..
#pragma unroll
          for (int i = 0; i < 4; i++) v[i] = lds16(at + 4096 + (16 * half + 8 * (i >> 1) + 2 * t4 + (i & 1)) * 128 + ((g ^ (2 * t4)) << 4));
#pragma unroll
          for (int wd = 0; wd < 4; wd++) {
            auto word = [&](int i) { return wd == 0 ? v[i].x : wd == 1 ? v[i].y : wd == 2 ? v[i].z : v[i].w; };
            const uint32_t bs[4][2] = {{codes_of<E4M3, 0>(word(0), word(1)), codes_of<E4M3, 0>(word(2), word(3))}, {codes_of<E4M3, 1>(word(0), word(1)), codes_of<E4M3, 1>(word(2), word(3))},
                                       {codes_of<E4M3, 2>(word(0), word(1)), codes_of<E4M3, 2>(word(2), word(3))}, {codes_of<E4M3, 3>(word(0), word(1)), codes_of<E4M3, 3>(word(2), word(3))}};
            if (ACROSS) {
#pragma unroll
              for (int i = 0; i < 2; i++) mma_bf16(o[0][2 * wd + i], bs[2 * i][0], bs[2 * i + 1][0], bs[2 * i][1], bs[2 * i + 1][1], pw[half][0], pw[half][1]);
              if (!PAIRED) {
#pragma unroll
                for (int i = 0; i < 2; i++) mma_bf16(o[0][2 * wd + i], bs[2 * i][0], bs[2 * i + 1][0], bs[2 * i][1], bs[2 * i + 1][1], pl[half][0], pl[half][1]);
              }
            } else {
              const int c = 2 * half % (NV / 2), d = (2 * half + 1) % (NV / 2);
#pragma unroll
              for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int i = 0; i < 4; i++) mma_bf16(o[mt][(4 * wd + i) % ON], pw[2 * mt][c], pw[2 * mt + 1][c], pw[2 * mt][d], pw[2 * mt + 1][d], bs[i][0], bs[i][1]);
#pragma unroll
              for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int i = 0; i < 4; i++) mma_bf16(o[mt][(4 * wd + i) % ON], pl[2 * mt][c], pl[2 * mt + 1][c], pl[2 * mt][d], pl[2 * mt + 1][d], bs[i][0], bs[i][1]);
            }
          }
        }
        __syncwarp();
        load_step(j + 2);
      }
    };
    if constexpr (NARROW) {
      if (!wide) coded_rows(std::false_type());
      else coded_rows(std::true_type());
    } else {
      coded_rows(std::true_type());
    }
    if (recent) {
      // ---- the rows behind the last whole block, 16 bf16 rows of this warp at a time.  Weights are two bf16 numbers each. ----
#pragma unroll 1
      for (int sub = 0; sub < 2; sub++) {
        const int r0 = whole + 64 * sub + 16 * warp, live = min(16, way.len - r0);
        at = mine + ((n_coded + sub) & 1) * A8_SLOT;
        cp_wait<1>();
        if (live <= 0) {
          cp_commit();
          continue;
        }
        float x[NR][4];   // score v: row 8 (v >> 1) + 2 t4 + (v & 1); across: row 8 v + g, v < 2
        constexpr int NB = ACROSS ? 2 : 4;
        if (ACROSS) {
          float acc[4] = {};
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const uint4 q = lds16(ROWS * 256 + g * A8_QS + t4 * 64 + i * 16), a = lds16(at + g * 256 + t4 * 64 + i * 16), c = lds16(at + (8 + g) * 256 + t4 * 64 + i * 16);
            mma_bf16(acc, a.x, c.x, a.y, c.y, q.x, q.y);
            mma_bf16(acc, a.z, c.z, a.w, c.w, q.z, q.w);
          }
          x[0][0] = acc[0], x[0][1] = acc[2], x[1][0] = acc[1], x[1][1] = acc[3];
        } else {
#pragma unroll
          for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int nt = 0; nt < 2; nt++) {
              float acc[4] = {};
#pragma unroll
              for (int i = 0; i < 4; i++) {
                const unsigned q = ROWS * 256 + (16 * mt + g) * A8_QS + t4 * 64 + i * 16;
                const uint4 w = lds16(at + (8 * nt + g) * 256 + t4 * 64 + i * 16), a = lds16(q), c = lds16(q + 8 * A8_QS);
                mma_bf16(acc, a.x, c.x, a.y, c.y, w.x, w.y);
                mma_bf16(acc, a.z, c.z, a.w, c.w, w.z, w.w);
              }
#pragma unroll
              for (int e = 0; e < 2; e++) x[2 * mt + e][2 * nt] = acc[2 * e], x[2 * mt + e][2 * nt + 1] = acc[2 * e + 1];
            }
        }
        uint32_t hi[NR][2], lo[NR][2];   // pairs of weights, and what their rounding left; across as above
#pragma unroll
        for (int e = 0; e < NR; e++) {
          float m = st[e].m, sum = 0.0f;
          bool seen[NB];
#pragma unroll
          for (int v = 0; v < NB; v++) {
            const int row = ACROSS ? 8 * v + g : 8 * (v >> 1) + 2 * t4 + (v & 1);
            seen[v] = row < live && r0 + row <= last[e];
            x[e][v] *= factor[e] != factor[e] ? NAN : p.scale_log2;
            if (seen[v]) m = fmaxf(m, x[e][v]);
          }
          m = row_max(m);
          const float least = m == -INFINITY ? 0.0f : m;
#pragma unroll
          for (int v = 0; v < NB; v++) {
            x[e][v] = seen[v] ? ex2(x[e][v] - least) : 0.0f;
            sum += x[e][v];
          }
          const float f = move(st[e], m);
          st[e].l += sum;
          if (__any_sync(0xffffffffu, f != 1.0f)) scale_row(e, f);
        }
#pragma unroll
        for (int e = 0; e < NR; e++)
#pragma unroll
          for (int i = 0; i < 2; i++) {
            const float a = ACROSS ? x[0][(2 * e + i) % 2] : x[e][2 * i], c = ACROSS ? x[1][(2 * e + i) % 2] : x[e][(2 * i + 1) % 4];
            two_of(a, c, hi[e][i], lo[e][i]);
          }
        if (ACROSS) {
#pragma unroll
          for (int i = 0; i < 2; i++) hi[0][i] = turn(PAIRED && t4 >= 2 ? lo[0][i] : hi[0][i]), lo[0][i] = turn(lo[0][i]);
        }
        // A weight of zero does not keep what is not a number out of a product: it is taken out, and given to the query rows that see it.
        uint4 v[2][4];   // [half of the lane's channels]: rows 2 t4, 2 t4 + 1, and eight further; channels 16 g ..
        auto load_v = [&]() {
#pragma unroll
          for (int part = 0; part < 2; part++)
#pragma unroll
            for (int i = 0; i < 4; i++) v[part][i] = lds16(at + 4096 + (8 * (i >> 1) + 2 * t4 + (i & 1)) * 256 + g * 32 + 16 * part);
        };
        load_v();
        bool bad = false;
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const uint4 w = v[i >> 2][i & 3];
          bad |= not_finite(w.x) | not_finite(w.x >> 16) | not_finite(w.y) | not_finite(w.y >> 16) | not_finite(w.z) | not_finite(w.z >> 16) | not_finite(w.w) | not_finite(w.w >> 16);
        }
        bad = __any_sync(0xffffffffu, bad);
        if (bad) {
#pragma unroll 1
          for (int row = 0; row < live; row++)
#pragma unroll
            for (int n = 0; n < 16; n++)
#pragma unroll
              for (int i = 0; i < (ACROSS ? 1 : 2); i++) {
                uint16_t w;
                asm volatile("ld.shared.u16 %0, [%1];" : "=h"(w) : "r"(base + at + 4096 + row * 256 + 2 * (ACROSS ? 16 * g + n : 32 * t4 + 16 * i + n)) : "memory");
                if (not_finite(w)) {
#pragma unroll
                  for (int e = 0; e < NR; e++)
                    if (r0 + row <= last[e]) {
                      if (ACROSS) o[0][(n >> 1) % ON][2 * (n & 1) + (e & 1)] += bf2f(w);
                      else o[e >> 1][n % ON][2 * (e & 1) + i] += bf2f(w);
                    }
                }
              }
          __syncwarp();
#pragma unroll 1
          for (int i = lane; i < 1024; i += 32) {
            uint32_t v;
            asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(base + at + 4096 + i * 4) : "memory");
            v = (not_finite(v) ? 0 : v & 0xffffu) | (not_finite(v >> 16) ? 0 : v & 0xffff0000u);
            asm volatile("st.shared.b32 [%0], %1;" ::"r"(base + at + 4096 + i * 4), "r"(v) : "memory");
          }
          __syncwarp();
          load_v();
        }
#pragma unroll
        for (int part = 0; part < 2; part++) {
#pragma unroll
          for (int k = 0; k < 4; k++) {
            auto word = [&](int i) { return k == 0 ? v[part][i].x : k == 1 ? v[part][i].y : k == 2 ? v[part][i].z : v[part][i].w; };
            const uint32_t b0 = __byte_perm(word(0), word(1), 0x5410), b1 = __byte_perm(word(2), word(3), 0x5410), c0 = __byte_perm(word(0), word(1), 0x7632),
                           c1 = __byte_perm(word(2), word(3), 0x7632);
            if (ACROSS) {
              mma_bf16(o[0][4 * part + k], b0, c0, b1, c1, hi[0][0], hi[0][1]);
              if (!PAIRED) mma_bf16(o[0][4 * part + k], b0, c0, b1, c1, lo[0][0], lo[0][1]);
            } else {
#pragma unroll
              for (int mt = 0; mt < MT; mt++) {
                float (&x0)[4] = o[mt][(8 * part + 2 * k) % ON], (&x1)[4] = o[mt][(8 * part + 2 * k + 1) % ON];
                mma_bf16(x0, hi[2 * mt][0], hi[2 * mt + 1][0], hi[2 * mt][1], hi[2 * mt + 1][1], b0, b1);
                mma_bf16(x0, lo[2 * mt][0], lo[2 * mt + 1][0], lo[2 * mt][1], lo[2 * mt + 1][1], b0, b1);
                mma_bf16(x1, hi[2 * mt][0], hi[2 * mt + 1][0], hi[2 * mt][1], hi[2 * mt + 1][1], c0, c1);
                mma_bf16(x1, lo[2 * mt][0], lo[2 * mt + 1][0], lo[2 * mt][1], lo[2 * mt + 1][1], c0, c1);
              }
            }
          }
        }
        __syncwarp();
        cp_commit();
      }
    }
    // ---- the four warps' shares of the segment ----
#pragma unroll
    for (int e = 0; e < NR; e++) {
#pragma unroll
      for (int off = ACROSS ? 4 : 1; off < (ACROSS ? 32 : 4); off <<= 1) st[e].l += __shfl_xor_sync(0xffffffffu, st[e].l, off);
      if (ACROSS ? g == 0 : t4 == 0) s_m[warp][row_of(e)] = st[e].m, s_l[warp][row_of(e)] = st[e].l;
    }
    __syncthreads();
    float* parts = reinterpret_cast<float*>(dyn8 + A8<ROWS>::q_bytes);   // a warp's first stage
    float* to = parts + warp * 2 * A8_SLOT / 4;
    auto share = [&](int e) {   // what this warp's O of a query row counts for
      const int r = row_of(e);
      const float M = fmaxf(fmaxf(s_m[0][r], s_m[1][r]), fmaxf(s_m[2][r], s_m[3][r]));
      return st[e].m == -INFINITY ? 0.0f : ex2(st[e].m - M);
    };
#pragma unroll
    for (int e = 0; e < (ACROSS ? 1 : NR); e++) {   // eight query rows at a time
      if (ACROSS) {
#pragma unroll
        for (int k = 0; k < 2; k++) {
          const float f = share(k);
#pragma unroll
          for (int n = 0; n < 8; n += 2)
            *reinterpret_cast<float4*>(to + A8<ROWS>::place(2 * t4 + k, 16 * g + 2 * n)) = make_float4(o[0][n][k] * f, o[0][n][2 + k] * f, o[0][n + 1][k] * f, o[0][n + 1][2 + k] * f);
        }
      } else if (8 * e < n_rows) {
        const float f = share(e);
        const int c = 2 * (e & 1);
#pragma unroll
        for (int n = 0; n < 16; n += 4) {
          float (&x0)[4] = o[e >> 1][n % ON], (&x1)[4] = o[e >> 1][(n + 1) % ON], (&x2)[4] = o[e >> 1][(n + 2) % ON], (&x3)[4] = o[e >> 1][(n + 3) % ON];
          *reinterpret_cast<float4*>(to + A8<ROWS>::place(g, 32 * t4 + n)) = make_float4(x0[c] * f, x1[c] * f, x2[c] * f, x3[c] * f);
          *reinterpret_cast<float4*>(to + A8<ROWS>::place(g, 32 * t4 + 16 + n)) = make_float4(x0[c + 1] * f, x1[c + 1] * f, x2[c + 1] * f, x3[c + 1] * f);
        }
      }
      __syncthreads();
      const int row = 8 * e + (tid >> 4), c = 8 * (tid & 15);   // 16 threads a row
      if (row < n_rows) {
        const float M = fmaxf(fmaxf(s_m[0][row], s_m[1][row]), fmaxf(s_m[2][row], s_m[3][row]));
        float L = 0.0f, O[8] = {};
#pragma unroll
        for (int w = 0; w < 4; w++) {
          L += s_l[w][row] * (s_m[w][row] == -INFINITY ? (s_l[w][row] == 0.0f ? 0.0f : 1.0f) : ex2(s_m[w][row] - M));   // (all NaN: the sum is NaN and stays)
          const float4* from = reinterpret_cast<const float4*>(parts + w * 2 * A8_SLOT / 4 + A8<ROWS>::place(tid >> 4, c));
          const float4 x = from[0], y = from[1];
          O[0] += x.x, O[1] += x.y, O[2] += x.z, O[3] += x.w, O[4] += y.x, O[5] += y.y, O[6] += y.z, O[7] += y.w;
          if (PAIRED) {
            const float4* more = reinterpret_cast<const float4*>(parts + w * 2 * A8_SLOT / 4 + A8<ROWS>::place((tid >> 4) + 4, c));
            const float4 x = more[0], y = more[1];
            O[0] += x.x, O[1] += x.y, O[2] += x.z, O[3] += x.w, O[4] += y.x, O[5] += y.y, O[6] += y.z, O[7] += y.w;
          }
        }
        if (whole_item) {
          const int rr = group * ROWS + row, t = rr / p.G, hq = h * p.G + rr % p.G;
          const int64_t out_row = ((int64_t)b * p.T + t) * Hq + hq;
          uint32_t w[4];
#pragma unroll
          for (int i = 0; i < 4; i++) w[i] = pack2(L == 0.0f ? 0.0f : O[2 * i] / L, L == 0.0f ? 0.0f : O[2 * i + 1] / L);
          *reinterpret_cast<uint4*>(p.out + out_row * 128 + c) = make_uint4(w[0], w[1], w[2], w[3]);
          if (p.lse && c == 0) p.lse[out_row] = L == 0.0f ? -INFINITY : M + log2f(L);
        } else if (p.cluster) {
          float4* rec = reinterpret_cast<float4*>(dyn8 + A8<ROWS>::q_bytes + e * 2 * A8_SLOT + A8_SLOT) + (tid >> 4) * 32 + (c >> 2);   // the second stage of warp e
          rec[0] = make_float4(O[0], O[1], O[2], O[3]), rec[1] = make_float4(O[4], O[5], O[6], O[7]);
          if (c == 0) s_M[row] = M, s_L[row] = L;
        } else {
          float4* rec = reinterpret_cast<float4*>(p.records + (2 * (int64_t)blockIdx.x + (way.tile == 0)) * (ROWS * 130) + row * 128 + c);
          rec[0] = make_float4(O[0], O[1], O[2], O[3]), rec[1] = make_float4(O[4], O[5], O[6], O[7]);
          if (c == 0) {
            float* tail = p.records + (2 * (int64_t)blockIdx.x + (way.tile == 0)) * (ROWS * 130) + ROWS * 128 + row;
            tail[0] = M, tail[ROWS] = L;
          }
        }
      }
      __syncthreads();
    }
  }
  if (p.cluster > 1) {   // the blocks of an item: each joins the rows that are its turn
    cluster_sync();
    const int item = (int)blockIdx.x / p.cluster, item_b = item / (int)items, item_h = item % (int)items / p.row_groups, item_group = item % p.row_groups;
    const int n_rows = min(ROWS, n_rows_all - item_group * ROWS);
    for (int row = (int)blockIdx.x % p.cluster + warp * p.cluster; row < n_rows; row += 4 * p.cluster) {   // a warp a row, four channels a lane
      const float* o = reinterpret_cast<const float*>(dyn8 + A8<ROWS>::q_bytes + (row >> 3) * 2 * A8_SLOT + A8_SLOT) + (row & 7) * 128 + 4 * lane;
      float m[8], l[8], M = -INFINITY, L = 0.0f;
      float4 x[8], O = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int i = 0; i < 8; i++) {
        if (i >= p.cluster) break;
        m[i] = remote(&s_M[row], i), l[i] = remote(&s_L[row], i), x[i] = remote4(o, i);
      }
#pragma unroll
      for (int i = 0; i < 8; i++)
        if (i < p.cluster) M = fmaxf(M, m[i]);
#pragma unroll
      for (int i = 0; i < 8; i++)
        if (i < p.cluster) {
          const float f = m[i] == -INFINITY ? 0.0f : ex2(m[i] - M);
          L += l[i] * f;
          if (m[i] != -INFINITY) O.x += x[i].x * f, O.y += x[i].y * f, O.z += x[i].z * f, O.w += x[i].w * f;   // (a block without rows of this item has not written any)
        }
      const int rr = item_group * ROWS + row, t = rr / p.G, hq = item_h * p.G + rr % p.G;
      const int64_t out_row = ((int64_t)item_b * p.T + t) * Hq + hq;
      const bool none = L == 0.0f;
      *reinterpret_cast<uint2*>(p.out + out_row * 128 + 4 * lane) = make_uint2(pack2(none ? 0.0f : O.x / L, none ? 0.0f : O.y / L), pack2(none ? 0.0f : O.z / L, none ? 0.0f : O.w / L));
      if (p.lse && lane == 0) p.lse[out_row] = none ? -INFINITY : M + log2f(L);
    }
    cluster_sync();   // no block ends while others read from it
  }
}

// A block per query row: the records of the blocks that share its item, in the order of the tiles.
template <int ROWS>
__global__ void __launch_bounds__(128) attend8_merge_kernel(const __grid_constant__ Attend8 p, int blocks) {
  // The lengths are read before the wait: this kernel starts once every block of the one before has triggered, which it does behind its own wait, and that one does not write them.
  __shared__ MergeShared shared;
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x & 31, Hq = p.c.H * p.G, hq = (int)(row % Hq), h = hq / p.G;
  const int64_t bt = row / Hq;
  const int t = (int)(bt % p.T), b = (int)(bt / p.T), r = t * p.G + hq % p.G;
  const int64_t items = (int64_t)p.c.H * p.row_groups;
  int64_t total = 0, before = 0;
  for (int b0 = 0; b0 < p.bs; b0 += 32) {
    const int tiles = b0 + lane < p.bs ? tiles8(p, len8(p, b0 + lane)) : 0;
    total += items * __reduce_add_sync(0xffffffffu, tiles), before += items * __reduce_add_sync(0xffffffffu, b0 + lane < b ? tiles : 0);
  }
  const int n = tiles8(p, len8(p, b));
  const int64_t first = before + ((int64_t)h * p.row_groups + r / ROWS) * n;
  const unsigned shares = (unsigned)min((int64_t)blocks, total);
  const bool apart = apart8(total, fewest8(p), shares);
  const int c0 = apart ? (int)first8(first, total, shares) : share_owner(first, total, shares), c1 = apart ? (int)first8(first + n, total, shares) - 1 : share_owner(first + n - 1, total, shares);
  pdl_wait();
  pdl_trigger();
  if (c0 == c1) return;   // written by its block
  const int cnt = c1 - c0 + 1, warp = threadIdx.x >> 5, q = r % ROWS;
  auto record = [&](int i) -> const float* { return p.records + (2 * (int64_t)(c0 + i) + (i == 0)) * (ROWS * 130); };
  if (cnt > 64) return merge_row<true>(shared, cnt, ROWS, q, record, p.out + row * 128, p.lse ? p.lse + row : nullptr);
  // Up to 64 records: all of them under way at once, a warp has every fourth, four channels a lane.
  float4 v[16], o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float m[2], l[2], f[2];
#pragma unroll
  for (int i = 0; i < 2; i++) {
    m[i] = lane + 32 * i < cnt ? record(lane + 32 * i)[ROWS * 128 + q] : -INFINITY;
    l[i] = lane + 32 * i < cnt ? record(lane + 32 * i)[ROWS * 129 + q] : 0.0f;
  }
#pragma unroll
  for (int k = 0; k < 16; k++) v[k] = 4 * k + warp < cnt ? *reinterpret_cast<const float4*>(record(4 * k + warp) + (int64_t)q * 128 + 4 * lane) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float M = fmaxf(m[0], m[1]);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, off));
#pragma unroll
  for (int i = 0; i < 2; i++) f[i] = m[i] == -INFINITY ? 0.0f : ex2(m[i] - M);
  float L = l[0] * f[0] + l[1] * f[1];   // (NaN stays, whatever it counts for)
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) L += __shfl_xor_sync(0xffffffffu, L, off);
#pragma unroll
  for (int k = 0; k < 16; k++) {
    const float w = __shfl_sync(0xffffffffu, f[k >> 3], (4 * k + warp) & 31);
    o.x += v[k].x * w, o.y += v[k].y * w, o.z += v[k].z * w, o.w += v[k].w * w;   // (a weight of zero too: what is not a number stays)
  }
  *reinterpret_cast<float4*>(&shared.o[warp][4 * lane]) = o;
  __syncthreads();
  const int c = threadIdx.x;
  const float O = (shared.o[0][c] + shared.o[1][c]) + (shared.o[2][c] + shared.o[3][c]);
  p.out[row * 128 + c] = f2bf(L == 0.0f ? 0.0f : O / L);
  if (p.lse && c == 0) p.lse[row] = L == 0.0f ? -INFINITY : M + log2f(L);
}

// Ranges per place on an SM.  SMs do not get the same share of HBM (with a range each the last ends a sixth after the average): of long ranges there are two, so that a fast place may take another.  (Below 1024
// blocks the shares are computed in 32 bits.)
int64_t a8_waves(int64_t most, int64_t slots) {
  return most / slots >= 48 ? 2 : 1;
}

// Query rows of an item.  Few tiles in all: eight, which has the shortest way through its code (B200, us, five tokens of five heads over 43 keys 6.1 | 9.4 with 32 rows, eight tokens of four heads over 1000
// keys 8.3 | 10.9); then as many as the KV head has, up to 32, because each item reads the cache again.
int a8_rows(int64_t heads, int64_t rows, int64_t tiles, int sms) {
  for (int n = 8; n < 32; n *= 2)
    if (rows <= n || heads * ((rows + n - 1) / n) * tiles <= 6 * sms) return n;
  return 32;
}
// Blocks of a cluster that share an item, so that one launch does and needs no scratch: where that leaves each at most three tiles.  0: ranges and a second launch.  B200, us, 701 keys of 8 KV heads of
// four queries 7.1, by two launches 8.5.
int a8_cluster(int64_t items, int64_t tiles, int64_t slots) {
  int64_t n = slots / items;
  n = n > 8 ? 8 : n < 1 ? 1 : n;
  n = n < tiles ? n : tiles;
  return (tiles + n - 1) / n <= 3 ? (int)n : 0;
}

template <bool E4M3, int ROWS, bool DENSE, bool PAIRED>
int launch_as(Attend8 p, cudaStream_t st) {
  p.row_groups = (p.T * p.G + ROWS - 1) / ROWS;
  const int64_t slots = (int64_t)A8<ROWS>::ctas * sm_count(), most = (int64_t)p.bs * p.c.H * p.row_groups * ((p.c.cap + A8_TILE - 1) / A8_TILE + 1);
  const int blocks = (int)(most < slots ? most : slots * a8_waves(most, slots));
  static PerDevice opted;
  if (const unsigned long long bit = first_on_device(opted)) {
    if (cudaFuncSetAttribute(attend8_kernel<E4M3, ROWS, DENSE, PAIRED>, cudaFuncAttributeMaxDynamicSharedMemorySize, A8<ROWS>::smem) != cudaSuccess)
      return fail(PK_ERR_CUDA, "cache8_attention: %s", cudaGetErrorString(cudaGetLastError()));
    mark_on_device(opted, bit);
  }
  StageTimer timer(ST_ATTENTION, st);
  const int64_t items = (int64_t)p.bs * p.c.H * p.row_groups;
  p.cluster = a8_cluster(items, most / items, slots);
  if (p.cluster) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(items * p.cluster)), cfg.blockDim = dim3(A8_THREADS), cfg.dynamicSmemBytes = A8<ROWS>::smem, cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension, attr[0].val.clusterDim.x = (unsigned)p.cluster, attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization, attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr, cfg.numAttrs = pdl_enabled() ? 2 : 1;
    cudaLaunchKernelEx(&cfg, attend8_kernel<E4M3, ROWS, DENSE, PAIRED>, p);
    return check_launch("cache8_attention");
  }
  launch_chain(attend8_kernel<E4M3, ROWS, DENSE, PAIRED>, dim3((unsigned)blocks), dim3(A8_THREADS), A8<ROWS>::smem, st, p);
  launch_chain(attend8_merge_kernel<ROWS>, dim3((unsigned)((int64_t)p.bs * p.T * p.c.H * p.G)), dim3(128), 0, st, p, blocks);
  return check_launch("cache8_attention", 2);
}

template <bool E4M3, int ROWS, bool PAIRED = false>
int launch(const Attend8& p, cudaStream_t st) {   // K and V of a row side by side, row after row: the copies' addresses are constants apart
  return p.c.c_l == 256 ? launch_as<E4M3, ROWS, true, PAIRED>(p, st) : launch_as<E4M3, ROWS, false, PAIRED>(p, st);
}
template <bool E4M3>
int launch_rows(const Attend8& p, int rows, cudaStream_t st) {
  if (p.T * p.G <= 4) return launch<E4M3, 8, true>(p, st);
  return rows == 8 ? launch<E4M3, 8>(p, st) : rows == 16 ? launch<E4M3, 16>(p, st) : launch<E4M3, 32>(p, st);
}

}  // namespace
}  // namespace pk

using namespace pk;

extern "C" int64_t pk_cache8_attention_workspace_bytes(int64_t bs, int64_t T, int64_t Hq, int64_t H, int64_t cap) {
  if (bs < 1 || T < 1 || T > 256 || H < 1 || Hq < H || cap < 0) return 0;
  const int64_t tiles = (cap + A8_TILE - 1) / A8_TILE + 1;
  const int rows = a8_rows(bs * H, T * (Hq / H), tiles, sm_count());
  const int64_t slots = (int64_t)(rows == 32 ? A8<32>::ctas : A8<8>::ctas) * sm_count(), most = bs * H * ((T * (Hq / H) + rows - 1) / rows) * tiles;
  const int64_t items = bs * H * ((T * (Hq / H) + rows - 1) / rows);
  if (a8_cluster(items, most / items, slots)) return 0;
  return 2 * (most < slots ? most : slots * a8_waves(most, slots)) * rows * 130 * 4;
}

extern "C" int pk_cache8_attention(const pk_tensor* queries, const pk_cache8* cache, const pk_tensor* lengths, float scale, const pk_tensor* out, const pk_tensor* lse, void* workspace,
                                   int64_t workspace_bytes, void* stream) {
  Attend8 p = {};
  if (const int rc = fill_cache8(&p.c, cache, false)) return rc;
  PK_CHECK_TENSOR(queries, PK_BF16, 4);
  PK_CHECK_TENSOR(lengths, PK_I32, 1);
  PK_CHECK_TENSOR(out, PK_BF16, 4);
  const int64_t bs = queries->shape[0], T = queries->shape[1], Hq = queries->shape[2], H = p.c.H;
  PK_REQUIRE(queries->shape[3] == 128 && row_tensor(queries), "queries must be bf16 [bs,T,Hq,128] with a unit inner stride, other strides that are multiples of 8, and 16-byte alignment");
  PK_REQUIRE(cache->codes->shape[0] == bs, "codes must be [bs,H,cap,2,128]");
  PK_REQUIRE(Hq % H == 0 && Hq >= H && Hq / H <= 128, "the query heads must be a multiple of the KV heads, at most 128 of them each");
  PK_REQUIRE(T <= 256, "at most 256 tokens");
  PK_REQUIRE(lengths->shape[0] == bs && is_contig(lengths), "lengths must be contiguous i32 [bs]");
  for (int i = 0; i < 4; i++) PK_REQUIRE(out->shape[i] == queries->shape[i], "out must have the shape of queries");
  PK_REQUIRE(is_contig(out) && aligned16(out->data), "out must be contiguous and 16-byte aligned");
  if (lse) {
    PK_CHECK_TENSOR(lse, PK_F32, 3);
    PK_REQUIRE(is_contig(lse) && lse->shape[0] == bs && lse->shape[1] == T && lse->shape[2] == Hq, "lse must be contiguous f32 [bs,T,Hq]");
    p.lse = (float*)lse->data;
  }
  PK_REQUIRE(bs < 65536 && bs * T * Hq < (1LL << 31) && bs * H * ((T * (Hq / H) + 7) / 8) < (1LL << 31) / (p.c.cap / A8_TILE + 2), "sizes out of range");
  p.scale_log2 = scale * 1.4426950408889634f;
  PK_REQUIRE(scale > 0.0f && p.scale_log2 <= 3.4e38f, "scale must be positive, and finite as a factor of log2 e");
  if (bs == 0 || T == 0) return PK_OK;
  const int64_t bytes = pk_cache8_attention_workspace_bytes(bs, T, Hq, H, p.c.cap);
  PK_REQUIRE(bytes == 0 || (workspace != nullptr && (reinterpret_cast<uintptr_t>(workspace) & 255) == 0), "workspace must be 256-byte aligned device memory");
  if (workspace_bytes < bytes) return fail(PK_ERR_WORKSPACE, "cache8_attention: workspace too small");
  p.q = (const uint16_t*)queries->data, p.q_b = queries->stride[0], p.q_t = queries->stride[1], p.q_h = queries->stride[2];
  p.lengths = (const int32_t*)lengths->data, p.bs = (int)bs, p.T = (int)T, p.G = (int)(Hq / H);
  p.out = (uint16_t*)out->data, p.records = (float*)workspace;
  const cudaStream_t st = (cudaStream_t)stream;
  const int rows = a8_rows(bs * H, p.T * p.G, (p.c.cap + A8_TILE - 1) / A8_TILE + 1, sm_count());
  return cache->codes->dtype == PK_E4M3 ? launch_rows<true>(p, rows, st) : launch_rows<false>(p, rows, st);
}
