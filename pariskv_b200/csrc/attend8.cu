// Attention of the last tokens of the sequences over the cache in 8 bits:  o = sum_j p_j v_j / sum_j p_j,  p_j = 2^((s_j - max s) scale log2 e),
//   s_j = ks (q . kc_j),  p_j v_j = (p_j vs) vc_j    with codes kc, vc of a row and the scales ks, vs of its block.
//
// HBM bounds a step: 256 bytes a row.  The products run on mma.sync with fp16 operands: a code is an fp16 number exactly (whole numbers: the byte becomes the last bits
// of 1024 + 128 + code, and 1152 is taken off), so is a query's value once its row has been scaled by a power of two; weights times value scales are rounded to 11 bits, scaled row by
// row by a power of two that follows the largest of them.
// The rows behind the last whole block come from `recent` as bf16, their weights as two bf16 numbers each.
//
// Every warp is by itself: 32 rows a step from global memory into its own stages of shared memory by cp.async, one step ahead.  The order of channels in Q K^T and of rows in P V is free, and
// chosen so that a lane's fragments of K are 32 consecutive codes of a row, and those of V 16 consecutive codes of four rows.
// Tiles of 128 rows, four warps of a block side by side, laid end to end over all (sample, KV head, row group) items, cut into equal ranges as in attend_few.cu.
#include "cache8.cuh"
#include "tiles.cuh"

namespace pk {
namespace {

constexpr int A8_TILE = 128, A8_THREADS = 128, A8_STAGES = 2;
constexpr int A8_ROWS = 16;                       // query rows of an item: those of one operand
constexpr int A8_STAGE = 8192;                    // 32 rows of K and V in codes, 16 in bf16
constexpr int A8_SLOT = A8_STAGE + 16;            // and the scales: K of the first and second 16 rows, V of them
constexpr int A8_SMEM = 4 * A8_STAGES * A8_SLOT;
constexpr int A8_CTAS = 3;
constexpr int A8_OS = 136;                        // floats between two rows of a warp's partial
static_assert(8 * A8_OS * 4 <= A8_STAGE, "a warp's partial of eight rows takes the place of a stage");

struct Attend8 {
  Cache8 c;
  const uint16_t* q;
  int64_t q_b, q_t, q_h;
  const int32_t* lengths;
  int bs, T, G, row_groups;
  float scale_log2;
  uint16_t* out;
  float *lse, *records;   // records: [2 * blocks][16 * 130]
};

__device__ __forceinline__ int len8(const Attend8& p, int b) { return (int)min((int64_t)max(p.lengths[b], 0), p.c.cap); }
__device__ __forceinline__ int tiles8(const Attend8& p, int len) {   // of an item: whole blocks, then the rows behind them
  const int whole = len >> p.c.shift << p.c.shift;
  return max(1, (whole + A8_TILE - 1) / A8_TILE + (whole < len));
}

// A warp's way through its steps: a tile of codes is one, a tile of 16-bit rows is two.
struct Way8 {
  int b, h, group, len, whole, n, tile, sub;
  int64_t left;   // tiles of the block's range that are left, this one included
  __device__ __forceinline__ void sample(const Attend8& p) { len = len8(p, b), whole = len >> p.c.shift << p.c.shift, n = tiles8(p, len); }
  __device__ __forceinline__ bool recent() const { return tile * A8_TILE >= whole && len > whole; }
  __device__ __forceinline__ int row0(int warp) const { return recent() ? whole + 32 * warp + 16 * sub : tile * A8_TILE + 32 * warp; }
  __device__ __forceinline__ int live(int warp) const {   // rows of this warp's step that are there
    return recent() ? max(0, min(16, len - row0(warp))) : max(0, min(32, whole - row0(warp)));
  }
  __device__ __forceinline__ bool last_of_item() const { return (recent() ? sub == 1 : true) && (tile == n - 1 || left == 1); }
  __device__ __forceinline__ void step(const Attend8& p) {
    if (recent() && sub == 0) {
      sub = 1;
      return;
    }
    sub = 0, left--;
    if (++tile < n) return;
    tile = 0;
    if (++group < p.row_groups) return;
    group = 0;
    if (++h < p.c.H) return;
    h = 0;
    if (++b < p.bs) sample(p);
  }
};

__device__ __forceinline__ void cp16(unsigned dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp4(unsigned dst, const void* src) { asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ uint4 lds16(unsigned at) {
  uint4 r;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(at) : "memory");
  return r;
}
__device__ __forceinline__ float lds4(unsigned at) {
  float r;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(r) : "r"(at) : "memory");
  return r;
}
__device__ __forceinline__ uint32_t half2_of(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Two codes (bytes lo, lo + 1 of w) as fp16 numbers.  Whole numbers come biased by 128.  e4m3: sign, exponent and significand in their places are 2^-8 of the value.
template <bool E4M3, int LO>
__device__ __forceinline__ uint32_t halves(uint32_t w) {
  uint32_t r;
  if (E4M3) {
    const uint32_t x = __byte_perm(w, 0, LO ? 0x3424 : 0x1404);   // each code is the upper byte of its half
    r = (x & 0x80008000u) | ((x & 0x7f007f00u) >> 1);
  } else {
    const uint32_t x = __byte_perm(w, 0x64646464u, LO ? 0x4342 : 0x4140);
    asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(0xe480e480u));   // 1024 + 128 + code - 1152
  }
  return r;
}
template <bool E4M3>
__device__ __forceinline__ uint32_t biased(uint32_t w) { return E4M3 ? w : w ^ 0x80808080u; }

// Running state of a lane's two rows (g and g + 8 of the item).
struct RowState {
  float m, l, u;        // largest score, sum of p (this lane's columns), largest p vs so far, all relative to m
  float up, down;       // 2^-E and 2^E: O is kept as 2^-E of what it stands for
};

// The weights of a step's columns: x[e][i] scores of row e (masked ones -inf), vs[i] the value scale of column i.  Leaves p vs 2^-E in x and scales what there is of O.
template <int N>
__device__ __forceinline__ void weigh(RowState (&st)[2], float (&o)[16][4], float (&x)[2][N], const float (&vs)[N], const float (&factor)[2]) {
  float f[2];
#pragma unroll
  for (int e = 0; e < 2; e++) {
    RowState& s = st[e];
    float mx = x[e][0];
#pragma unroll
    for (int i = 1; i < N; i++) mx = fmaxf(mx, x[e][i]);
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    const float m = fmaxf(s.m, mx), least = m == -INFINITY ? 0.0f : m;
    f[e] = s.m == -INFINITY ? 0.0f : m > s.m ? ex2((s.m - m) * factor[e]) : 1.0f;
    float sum = 0.0f, top = 0.0f;
#pragma unroll
    for (int i = 0; i < N; i++) {
      const bool seen = x[e][i] != -INFINITY;   // (a NaN is seen)
      const float y = seen ? ex2((x[e][i] - least) * factor[e]) : 0.0f;
      sum += y;
      x[e][i] = seen ? y * vs[i] : 0.0f;   // (the scale of a block that it does not see may be NaN)
      top = fmaxf(top, x[e][i]);
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    s.m = m, s.l = s.l * f[e] + sum;
    const float before = s.u * f[e];
    s.u = fmaxf(before, top);
    const float t = s.u * s.up;
    if (s.u > 0.0f && !(t >= 0.0625f && t <= 256.0f)) {   // (the same for the four lanes of a row)
      const unsigned ex = min(__float_as_uint(s.u) >> 23, 252u);
      s.up = __uint_as_float((254u - ex) << 23);
      f[e] = before == 0.0f ? 0.0f : f[e] * s.up * s.down;
      s.down = ex == 0 ? __uint_as_float(1u << 22) : __uint_as_float(ex << 23);
    }
#pragma unroll
    for (int i = 0; i < N; i++) x[e][i] *= s.up;
  }
  if (__any_sync(0xffffffffu, f[0] != 1.0f || f[1] != 1.0f)) {
#pragma unroll
    for (int n = 0; n < 16; n++) o[n][0] *= f[0], o[n][1] *= f[0], o[n][2] *= f[1], o[n][3] *= f[1];
  }
}

template <bool E4M3>
__global__ void __launch_bounds__(A8_THREADS, A8_CTAS) attend8_kernel(const __grid_constant__ Attend8 p) {
  extern __shared__ __align__(128) unsigned char dyn[];
  __shared__ float s_m[4][16], s_l[4][16], s_u[4][16];
  __shared__ TilePlan s_plan;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  pdl_wait();
  pdl_trigger();
  const int blocks = (int)gridDim.x;
  const int64_t items = (int64_t)p.c.H * p.row_groups;
  if (warp == 0) {
    const TilePlan w = tile_plan(p.bs, blockIdx.x, (unsigned)blocks, [&](int b) -> int64_t { return b < p.bs ? items * tiles8(p, len8(p, b)) : 0; });
    if (lane == 0) s_plan = w;
  }
  __syncthreads();
  const TilePlan plan = s_plan;
  const unsigned shares = (unsigned)min((int64_t)blocks, plan.total);
  if (blockIdx.x >= shares) return;
  Way8 way;
  {
    const int64_t first = share_begin(plan.total, blockIdx.x, shares);
    way.left = share_begin(plan.total, blockIdx.x + 1, shares) - first;
    way.b = plan.sample, way.sub = 0;
    way.sample(p);
    const int64_t at = first - plan.before;
    const int64_t item = at / way.n;
    way.tile = (int)(at % way.n), way.h = (int)(item / p.row_groups), way.group = (int)(item % p.row_groups);
  }
  const unsigned mine = smem_addr(dyn) + warp * A8_STAGES * A8_SLOT;
  // One step's rows on their way.  A chunk of 16 bytes lies where its row's number moves it, so that the reads below fall into all banks.
  auto load = [&](const Way8& w, int slot) {
    const unsigned to = mine + slot * A8_SLOT;
    const int live = w.live(warp), row0 = w.row0(warp);
    if (live > 0) {
      if (w.recent()) {
        const uint16_t* src = p.c.recent + w.b * p.c.r_b + w.h * p.c.r_h + (lane >> 4) * p.c.r_kv + (lane & 15) * 8;
#pragma unroll
        for (int i = 0; i < 16; i++) cp16(to + (lane >> 4) * 4096 + i * 256 + (lane & 15) * 16, src + (int64_t)((i < live ? row0 + i : row0) % p.c.R) * p.c.r_l, i < live);
      } else {
        const int c = lane & 7, kv = lane >> 3 & 1, odd = lane >> 4;
        const uint8_t* src = p.c.codes + w.b * p.c.c_b + w.h * p.c.c_h + kv * p.c.c_kv + (int64_t)row0 * p.c.c_l + c * 16;
#pragma unroll
        for (int i = 0; i < 16; i++) {
          const int r = 2 * i + odd;
          cp16(to + kv * 4096 + r * 128 + ((c ^ (kv ? r & 6 : r & 1)) << 4), src + (r < live ? r : 0) * p.c.c_l, r < live);
        }
        if (lane < 4) {
          const int j = min(row0 + 16 * (lane & 1), w.whole - 1) >> p.c.shift;
          cp4(to + A8_STAGE + 4 * lane, p.c.scales + w.b * p.c.s_b + w.h * p.c.s_h + (int64_t)j * p.c.s_j + (lane >> 1) * p.c.s_kv);
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  Way8 ahead = way;
  int slot = 0;
#pragma unroll
  for (int i = 0; i < A8_STAGES - 1; i++) {
    if (ahead.left > 0) load(ahead, i), ahead.step(p);
    else asm volatile("cp.async.commit_group;" ::: "memory");
  }
  const int n_rows_all = p.T * p.G, Hq = p.c.H * p.G;
  while (way.left > 0) {
    // ---- a segment: consecutive tiles of one item ----
    const int b = way.b, h = way.h, group = way.group, seg_first = way.tile;
    const bool whole_item = way.tile == 0 && way.left >= way.n;
    const int n_rows = min(A8_ROWS, n_rows_all - group * A8_ROWS);
    uint32_t qa[8][4];
    float factor[2];   // of the scores of codes: what the query row was scaled by, and log2 e / sqrt d
    int last[2];       // the last row that a query row sees
    const uint16_t* q_row[2];
#pragma unroll
    for (int e = 0; e < 2; e++) {
      const int r = group * A8_ROWS + min(8 * e + g, n_rows - 1), t = r / p.G;
      last[e] = p.lengths[b] > p.c.cap ? (int)p.c.cap - p.T + t : p.lengths[b] - p.T + t;
      q_row[e] = p.q + b * p.q_b + (int64_t)t * p.q_t + (int64_t)(h * p.G + r % p.G) * p.q_h + 32 * t4;
      uint4 x[4];
#pragma unroll
      for (int i = 0; i < 4; i++) x[i] = *reinterpret_cast<const uint4*>(q_row[e] + 8 * i);
      const uint32_t* xw = reinterpret_cast<const uint32_t*>(x);
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 16; i++) top = __vmaxu2(top, xw[i] & 0x7fff7fffu);
      top = max(top & 0xffffu, top >> 16);
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // the largest of the row becomes a number from 1 to 2; a row with an infinity or NaN becomes NaN
      const unsigned ex = max(min(top >> 7, 252u), 2u);
      const bool fine = top < 0x7f80u;
      const float up = fine ? __uint_as_float((254u - ex) << 23) : NAN;
#pragma unroll
      for (int i = 0; i < 16; i++)   // word i: channels 2 i, 2 i + 1 of this lane's 32
        qa[i >> 1][2 * (i & 1) + e] = half2_of(__uint_as_float(xw[i] << 16) * up, __uint_as_float(xw[i] & 0xffff0000u) * up);
      factor[e] = fine ? __uint_as_float(ex << 23) * p.scale_log2 : NAN;
    }
    if (E4M3) factor[0] *= 256.0f, factor[1] *= 256.0f;
    float o[16][4] = {};
    RowState st[2];
#pragma unroll
    for (int e = 0; e < 2; e++) st[e] = {-INFINITY, 0.0f, 0.0f, 1.0f, 1.0f};
    bool end = false;
    unsigned at;
    do {
      if (ahead.left > 0) load(ahead, (slot + A8_STAGES - 1) % A8_STAGES), ahead.step(p);
      else asm volatile("cp.async.commit_group;" ::: "memory");
      asm volatile("cp.async.wait_group %0;" ::"n"(A8_STAGES - 1) : "memory");
      __syncwarp();
      at = mine + slot * A8_SLOT;
      const int live = way.live(warp), row0 = way.row0(warp);
      if (live > 0 && !way.recent()) {
        float ks[2], vs2[2];
#pragma unroll
        for (int i = 0; i < 2; i++) ks[i] = lds4(at + A8_STAGE + 4 * i), vs2[i] = lds4(at + A8_STAGE + 8 + 4 * i);
        float x[2][8], vs[8];
#pragma unroll
        for (int nt = 0; nt < 4; nt++) {
          const int key = 8 * nt + g;
          const uint4 w0 = lds16(at + key * 128 + (((2 * t4) ^ (key & 1)) << 4)), w1 = lds16(at + key * 128 + (((2 * t4 + 1) ^ (key & 1)) << 4));
          const uint32_t w[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
          float acc[2][4] = {};
#pragma unroll
          for (int s = 0; s < 8; s++) {
            const uint32_t c = biased<E4M3>(w[s]);
            mma_f16(acc[s & 1], qa[s], halves<E4M3, 0>(c), halves<E4M3, 1>(c));
          }
#pragma unroll
          for (int i = 0; i < 4; i++) x[i >> 1][2 * nt + (i & 1)] = (acc[0][i] + acc[1][i]) * ks[nt >> 1];
          vs[2 * nt] = vs[2 * nt + 1] = vs2[nt >> 1];
        }
        const int lim = min(last[0], last[1]);
        if (__any_sync(0xffffffffu, live < 32 || row0 + 31 > lim)) {
#pragma unroll
          for (int e = 0; e < 2; e++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
              const int r = 8 * (i >> 1) + 2 * t4 + (i & 1);
              if (r >= live || row0 + r > last[e]) x[e][i] = -INFINITY;
            }
        }
        weigh<8>(st, o, x, vs, factor);
#pragma unroll
        for (int ks2 = 0; ks2 < 2; ks2++) {
          uint32_t pa[4];
#pragma unroll
          for (int i = 0; i < 2; i++)
#pragma unroll
            for (int e = 0; e < 2; e++) pa[2 * i + e] = half2_of(x[e][4 * ks2 + 2 * i], x[e][4 * ks2 + 2 * i + 1]);
          uint32_t v[4][4];
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const int key = 16 * ks2 + 8 * (i >> 1) + 2 * t4 + (i & 1);
            const uint4 w = lds16(at + 4096 + key * 128 + ((g ^ (key & 6)) << 4));
            v[i][0] = w.x, v[i][1] = w.y, v[i][2] = w.z, v[i][3] = w.w;
          }
#pragma unroll
          for (int wd = 0; wd < 4; wd++) {
            uint32_t pr[2][2];   // [rows of the first or second eight][channels 0, 1 or 2, 3 of the word]: two rows' codes of a channel side by side
#pragma unroll
            for (int i = 0; i < 2; i++) {
              const uint32_t a = biased<E4M3>(v[2 * i][wd]), c = biased<E4M3>(v[2 * i + 1][wd]);
              pr[i][0] = __byte_perm(a, c, 0x5140), pr[i][1] = __byte_perm(a, c, 0x7362);
            }
            mma_f16(o[4 * wd], pa, halves<E4M3, 0>(pr[0][0]), halves<E4M3, 0>(pr[1][0]));
            mma_f16(o[4 * wd + 1], pa, halves<E4M3, 1>(pr[0][0]), halves<E4M3, 1>(pr[1][0]));
            mma_f16(o[4 * wd + 2], pa, halves<E4M3, 0>(pr[0][1]), halves<E4M3, 0>(pr[1][1]));
            mma_f16(o[4 * wd + 3], pa, halves<E4M3, 1>(pr[0][1]), halves<E4M3, 1>(pr[1][1]));
          }
        }
      } else if (live > 0) {
        // ---- 16 rows in bf16 ----
        float x[2][4];
        const float raw[2] = {p.scale_log2 / factor[0], p.scale_log2 / factor[1]};   // scores in the units of the codes' ones
#pragma unroll
        for (int nt = 0; nt < 2; nt++) {
          float acc[4] = {};
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const uint4 w = lds16(at + (8 * nt + g) * 256 + t4 * 64 + i * 16);
            const uint4 a = *reinterpret_cast<const uint4*>(q_row[0] + 8 * i), c = *reinterpret_cast<const uint4*>(q_row[1] + 8 * i);
            const uint32_t f0[4] = {a.x, c.x, a.y, c.y}, f1[4] = {a.z, c.z, a.w, c.w};
            mma_bf16(acc, f0, w.x, w.y);
            mma_bf16(acc, f1, w.z, w.w);
          }
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const int r = 8 * nt + 2 * t4 + (i & 1), e = i >> 1;
            x[e][2 * nt + (i & 1)] = r < live && row0 + r <= last[e] ? acc[i] * raw[e] : -INFINITY;
          }
        }
        const float one = E4M3 ? 0.00390625f : 1.0f;   // O of e4m3 codes is kept as 2^-8 of what it stands for
        const float vs[4] = {one, one, one, one};
        weigh<4>(st, o, x, vs, factor);
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
          for (int e = 0; e < 2; e++) {
            const float a = x[e][2 * i], c = x[e][2 * i + 1];
            const uint32_t w = pack2(a, c);
            hi[2 * i + e] = w;
            lo[2 * i + e] = pack2(a - __uint_as_float(w << 16), c - __uint_as_float(w & 0xffff0000u));
          }
        uint32_t v[4][8];
        bool bad = false;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int key = 8 * (i >> 1) + 2 * t4 + (i & 1);
          const uint4 w0 = lds16(at + 4096 + key * 256 + g * 32), w1 = lds16(at + 4096 + key * 256 + g * 32 + 16);
          v[i][0] = w0.x, v[i][1] = w0.y, v[i][2] = w0.z, v[i][3] = w0.w, v[i][4] = w1.x, v[i][5] = w1.y, v[i][6] = w1.z, v[i][7] = w1.w;
#pragma unroll
          for (int k = 0; k < 8; k++) bad |= not_finite(v[i][k]) | not_finite(v[i][k] >> 16);
        }
        bad = __any_sync(0xffffffffu, bad);
        if (bad) {   // a weight of zero does not keep what is not a number out of a product: it is taken out, and given to the query rows that see it
#pragma unroll
          for (int i = 0; i < 4; i++)
#pragma unroll
            for (int k = 0; k < 8; k++) v[i][k] = (not_finite(v[i][k]) ? 0 : v[i][k] & 0xffffu) | (not_finite(v[i][k] >> 16) ? 0 : v[i][k] & 0xffff0000u);
        }
#pragma unroll
        for (int k = 0; k < 8; k++) {
          const uint32_t b0 = __byte_perm(v[0][k], v[1][k], 0x5410), b1 = __byte_perm(v[2][k], v[3][k], 0x5410), c0 = __byte_perm(v[0][k], v[1][k], 0x7632),
                         c1 = __byte_perm(v[2][k], v[3][k], 0x7632);
          mma_bf16(o[2 * k], hi, b0, b1);
          mma_bf16(o[2 * k], lo, b0, b1);
          mma_bf16(o[2 * k + 1], hi, c0, c1);
          mma_bf16(o[2 * k + 1], lo, c0, c1);
        }
        if (bad) {
          for (int r = 0; r < live; r++)
#pragma unroll
            for (int n = 0; n < 16; n++)
#pragma unroll
              for (int i = 0; i < 2; i++) {   // column n of the two n-tile columns 2 t4, 2 t4 + 1 of this lane: channel 32 t4 + 16 i + n
                uint16_t w;
                asm volatile("ld.shared.u16 %0, [%1];" : "=h"(w) : "r"(at + 4096 + r * 256 + 2 * (32 * t4 + 16 * i + n)) : "memory");
                if (not_finite(w)) {
                  if (row0 + r <= last[0]) o[n][i] += bf2f(w);
                  if (row0 + r <= last[1]) o[n][2 + i] += bf2f(w);
                }
              }
        }
      }
      __syncwarp();
      end = way.last_of_item();
      way.step(p);
      slot = (slot + 1) % A8_STAGES;
    } while (!end);
    // ---- the four warps' shares of the segment ----
#pragma unroll
    for (int e = 0; e < 2; e++) {
      st[e].l += __shfl_xor_sync(0xffffffffu, st[e].l, 1);
      st[e].l += __shfl_xor_sync(0xffffffffu, st[e].l, 2);
      if (t4 == 0) s_m[warp][8 * e + g] = st[e].m == -INFINITY ? -INFINITY : st[e].m * factor[e], s_l[warp][8 * e + g] = st[e].l, s_u[warp][8 * e + g] = st[e].down * (E4M3 ? 256.0f : 1.0f);
    }
    __syncthreads();
    float* rec = whole_item ? nullptr : p.records + (2 * (int64_t)blockIdx.x + (seg_first == 0)) * (A8_ROWS * 130);
    const unsigned part = at - smem_addr(dyn);   // the stage of the segment's last step: the same of every warp
    float* to = reinterpret_cast<float*>(dyn + part) + g * A8_OS + 32 * t4;
#pragma unroll
    for (int e = 0; e < 2; e++) {
      if (8 * e < n_rows) {
        const int r = 8 * e + g;
        const float M = fmaxf(fmaxf(s_m[0][r], s_m[1][r]), fmaxf(s_m[2][r], s_m[3][r]));
        const float f = s_m[warp][r] == -INFINITY ? 0.0f : ex2(s_m[warp][r] - M);
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
          for (int n = 0; n < 16; n += 4)
            *reinterpret_cast<float4*>(to + 16 * i + n) = make_float4(o[n][2 * e + i] * f * s_u[warp][r], o[n + 1][2 * e + i] * f * s_u[warp][r], o[n + 2][2 * e + i] * f * s_u[warp][r],
                                                                       o[n + 3][2 * e + i] * f * s_u[warp][r]);
      }
      __syncthreads();
      if (8 * e < n_rows) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const int row = 8 * e + i;
          if (row < n_rows) {
            const float M = fmaxf(fmaxf(s_m[0][row], s_m[1][row]), fmaxf(s_m[2][row], s_m[3][row]));
            float L = 0.0f, O = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; w++) {
              L += s_l[w][row] * (s_m[w][row] == -INFINITY ? (s_l[w][row] == 0.0f ? 0.0f : 1.0f) : ex2(s_m[w][row] - M));   // (all NaN: the sum is NaN and stays)
              O += reinterpret_cast<const float*>(dyn + (part % (A8_STAGES * A8_SLOT)) + w * A8_STAGES * A8_SLOT)[i * A8_OS + tid];
            }
            const int rr = group * A8_ROWS + row, t = rr / p.G, hq = h * p.G + rr % p.G;
            if (whole_item) {
              const int64_t out_row = ((int64_t)b * p.T + t) * Hq + hq;
              p.out[out_row * 128 + tid] = f2bf(L == 0.0f ? 0.0f : O / L);
              if (p.lse && tid == 0) p.lse[out_row] = L == 0.0f ? -INFINITY : M + log2f(L);
            } else {
              rec[row * 128 + tid] = O;
              if (tid == 0) rec[A8_ROWS * 128 + row] = M, rec[A8_ROWS * 129 + row] = L;
            }
          }
        }
      }
      __syncthreads();
    }
  }
}

// A block per query row: the records of the blocks that share its item, in the order of the tiles.
__global__ void __launch_bounds__(128) attend8_merge_kernel(const __grid_constant__ Attend8 p, int blocks) {
  pdl_wait();
  pdl_trigger();
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
  const int64_t first = before + ((int64_t)h * p.row_groups + r / A8_ROWS) * n;
  const unsigned shares = (unsigned)min((int64_t)blocks, total);
  const int c0 = share_owner(first, total, shares), c1 = share_owner(first + n - 1, total, shares);
  if (c0 == c1) return;   // written by its block
  merge_row(shared, c1 - c0 + 1, A8_ROWS, r % A8_ROWS, [&](int i) { return p.records + (2 * (int64_t)(c0 + i) + (i == 0)) * (A8_ROWS * 130); }, p.out + row * 128,
            p.lse ? p.lse + row : nullptr);
}

template <bool E4M3>
int launch(const Attend8& p, cudaStream_t st) {
  const int64_t slots = (int64_t)A8_CTAS * sm_count(), most = (int64_t)p.bs * p.c.H * p.row_groups * ((p.c.cap + A8_TILE - 1) / A8_TILE + 1);
  const int blocks = (int)(most < slots ? most : slots);
  static PerDevice opted;
  if (const unsigned long long bit = first_on_device(opted)) {
    if (cudaFuncSetAttribute(attend8_kernel<E4M3>, cudaFuncAttributeMaxDynamicSharedMemorySize, A8_SMEM) != cudaSuccess)
      return fail(PK_ERR_CUDA, "cache8_attention: %s", cudaGetErrorString(cudaGetLastError()));
    mark_on_device(opted, bit);
  }
  StageTimer timer(ST_ATTENTION, st);
  launch_chain(attend8_kernel<E4M3>, dim3((unsigned)blocks), dim3(A8_THREADS), A8_SMEM, st, p);
  launch_chain(attend8_merge_kernel, dim3((unsigned)((int64_t)p.bs * p.T * p.c.H * p.G)), dim3(128), 0, st, p, blocks);
  return check_launch("cache8_attention", 2);
}

}  // namespace
}  // namespace pk

using namespace pk;

extern "C" int64_t pk_cache8_attention_workspace_bytes(int64_t bs, int64_t T, int64_t Hq, int64_t H, int64_t cap) {
  if (bs < 1 || T < 1 || T > 256 || H < 1 || Hq < H || cap < 0) return 0;
  return 2 * (int64_t)A8_CTAS * sm_count() * A8_ROWS * 130 * 4;
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
  PK_REQUIRE(bs < 65536 && bs * T * Hq < (1LL << 31), "sizes out of range");
  p.scale_log2 = scale * 1.4426950408889634f;
  PK_REQUIRE(scale > 0.0f && p.scale_log2 <= 3.4e38f, "scale must be positive, and finite as a factor of log2 e");
  if (bs == 0 || T == 0) return PK_OK;
  PK_REQUIRE(workspace != nullptr && (reinterpret_cast<uintptr_t>(workspace) & 255) == 0, "workspace must be 256-byte aligned device memory");
  if (workspace_bytes < pk_cache8_attention_workspace_bytes(bs, T, Hq, H, p.c.cap)) return fail(PK_ERR_WORKSPACE, "cache8_attention: workspace too small");
  p.q = (const uint16_t*)queries->data, p.q_b = queries->stride[0], p.q_t = queries->stride[1], p.q_h = queries->stride[2];
  p.lengths = (const int32_t*)lengths->data, p.bs = (int)bs, p.T = (int)T, p.G = (int)(Hq / H), p.row_groups = (int)((T * p.G + A8_ROWS - 1) / A8_ROWS);
  p.out = (uint16_t*)out->data, p.records = (float*)workspace;
  return cache->codes->dtype == PK_E4M3 ? launch<true>(p, (cudaStream_t)stream) : launch<false>(p, (cudaStream_t)stream);
}
