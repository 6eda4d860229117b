// y = x W^T for a few tokens, W of 4-bit codes c with a scale s (and an offset m) per row and group of columns:
//   W = (c - 8) s, or c s + m;   y = sum over groups q of  s_q (sum c x - 8 sum x), or s_q sum c x + m_q sum x
// The products run on the tensor cores (mma.sync), 16 rows of W by 8 columns, in one of two forms:
//   whole numbers, for one token.  x = e (d0 + d1 / 2^7 + .. + d7 / 2^49) per group, e a power of two, the digits of 8 bits: the eight columns of a
//     product, exact sums.  A value that is 2^-48 of its group's largest still has all of its bits, one below 2^-55 of it counts as zero; no smaller
//     unit than 2^-126 is used.  A word of eight codes costs three instructions of the integer unit.  The sums start from 2^23 + 2^22 - 8 sum d
//     in the bits of a float, so that their bits are that float's: e and s follow in fp32.
//   bf16, a column a token.  A code becomes one by its bits, 0x4300 | c = 128 + c, less 136 (128 with offsets), which is exact: seven instructions of
//     the integer unit and four subtractions a word, and a weight of zero adds nothing whatever it meets.
// The integer unit, not the tensor cores, is what both spend most on; what each takes stands at w4_plan().
//
// Bounded by the bytes of W.  Sixteen rows are a unit; a box is 256 (or 512) of its columns, 2 KB pieces that TMA brings with the 128-byte swizzle, a warp's
// share of a stage of sixteen boxes.  A lane reads a word of 8 codes of rows g and g + 8 and 8 digits per 32 columns and product; the digits
// lie in shared memory in the order of the codes' bits.  Where rows are long sixteen warps share a unit, where they are short as many units
// share a stage; the warps' sums meet in shared memory once per unit.  Gated: eight rows of the gate and the eight of the up product they
// meet are a unit.
#include <type_traits>

#include "attend.cuh"
#include "tma.cuh"

namespace pk {
namespace {

constexpr int W4_WARPS = 16, W4_THREADS = 32 * W4_WARPS + 64;   // the warps of the products, one that makes the copies, one that adds the warps' sums
constexpr int W4_PIECE = 2048;                  // 256 columns of 16 rows
// Stages at most; units whose warps' sums are kept, with NT times eight columns.
constexpr int W4_STAGES_MAX = 6;
__host__ __device__ constexpr int w4_sums(int nt) { return nt == 1 ? 4 : 2; }
constexpr int W4_DIGITS = 8;                    // of a value in whole numbers
constexpr uint32_t W4_BIAS = 0x4b400000u;       // the float 2^23 + 2^22: adding a whole number below 2^22 to its bits adds it to the float
constexpr int W4_LONG = 8;                       // stages of 64 KB per SM from which on boxes are of 512 columns
constexpr int W4_WAIT_LIMIT = 100000;
constexpr int W4_SMEM = 227 * 1024 - 512;   // of a block; 512 bytes of barriers

struct W4Params {
  const uint8_t* w;
  const uint16_t *scales, *offsets, *x;
  int64_t x_t;
  uint16_t* out;
  int n_out, I, T, group_log, gated;
  int units, boxes, kw_log;      // boxes of a unit and slice; 1 << kw_log warps on a unit
  int stages;
  int slices;                    // parts of the columns, where x does not fit at once
  int pitch;                     // bytes from one column of digits to the next
  int groups_smem;               // groups of a slice
  float* partial;                // [units][32][4 NT]: sums of the slices before
  bool early;
};

__device__ __forceinline__ void mma_codes(uint32_t (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void tma_load2(unsigned dst, const CUtensorMap* map, int c0, int c1, unsigned mb) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst), "l"(map), "r"(c0),
               "r"(c1), "r"(mb)
               : "memory");
}
__device__ __forceinline__ void mma_bf16(uint32_t (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// codes 0 and 4 of a word as bf16 128 + c
__device__ __forceinline__ uint32_t code_pair(uint32_t w, uint32_t mask, uint32_t magic) {   // one instruction: both constants in registers
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(w), "r"(mask), "r"(magic));
  return r;
}

// two bf16 less another: whole numbers below 256, exact
__device__ __forceinline__ uint32_t less2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// Whole numbers: what a group's sum of a column starts from and is scaled by.
struct W4Column {
  uint32_t start;   // W4_BIAS - 8 sum d, or W4_BIAS
  float e;          // e / 2^(7 digit)
};

// WHOLE: the form; NT: its columns in eights; SUB: pieces of 256 columns in a box
template <bool WHOLE, int NT, int SUB>
__global__ void __launch_bounds__(W4_THREADS, 1) gemv_w4_kernel(const __grid_constant__ CUtensorMap map, const __grid_constant__ W4Params p) {
  constexpr int W4_BOX = SUB * W4_PIECE, W4_STAGE = W4_WARPS * W4_BOX, SUMS = w4_sums(NT), E = 2 * SUB, PER = WHOLE ? W4_DIGITS : 1;   // E: scales of a row that a lane holds; PER: columns of a token
  constexpr int BYTES = WHOLE ? 1 : 2;   // of a value of x in shared memory
  extern __shared__ unsigned char dyn[];
  __shared__ __align__(8) unsigned long long bars[2 * W4_STAGES_MAX + 2 * SUMS];
  __shared__ volatile int s_dead;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  const unsigned base = (smem_addr(dyn) + 1023) & ~1023u, full = smem_addr(bars), empty = full + 8 * W4_STAGES_MAX, sums_full = empty + 8 * W4_STAGES_MAX, sums_empty = sums_full + 8 * SUMS;
  unsigned char* at_base = dyn + (base - smem_addr(dyn));
  float* s_red = reinterpret_cast<float*>(at_base + p.stages * W4_STAGE);          // [SUMS][NT][16 warps][32 lanes][4]
  float* s_out = s_red + SUMS * W4_WARPS * 32 * 4 * NT;                             // [NT][32 lanes][4]: of one unit
  W4Column* s_col = reinterpret_cast<W4Column*>(s_out + 128 * NT);                  // [groups][8 NT] (whole numbers)
  float* s_x = reinterpret_cast<float*>(s_col + (WHOLE ? p.groups_smem * 8 * NT : 0));   // [groups][8 NT]: sum of x, the column's part (with offsets)
  unsigned char* s_dig = reinterpret_cast<unsigned char*>(s_x + (p.offsets ? p.groups_smem * 8 * NT : 0));   // x: [columns, and one of zeros if there are no eights of them][pitch]
  const int kw = 1 << p.kw_log, per_stage = W4_WARPS >> p.kw_log;                   // warps on a unit, units of a stage
  const int steps = (p.boxes + kw - 1) >> p.kw_log;                                 // stages of a unit
  const int sets = (p.units + per_stage - 1) / per_stage, mine = ((int)gridDim.x - 1 - (int)blockIdx.x + sets) / (int)gridDim.x;   // sets of units that share stages
  if (tid == 0) {
    for (int i = 0; i < p.stages; i++) mbar_init(full + 8 * i, 1), mbar_init(empty + 8 * i, W4_WARPS);
    for (int i = 0; i < SUMS; i++) mbar_init(sums_full + 8 * i, W4_WARPS), mbar_init(sums_empty + 8 * i, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    s_dead = 0;
  }
  if (tid == 32 * W4_WARPS) tma_prefetch_map(&map);
  __syncthreads();
  bool dead = false;   // a wait has run out: no more waiting, the outputs come out as NaN
  auto wait = [&](unsigned mb, unsigned parity) {
    for (int it = 0; !dead; it++) {
      if (mbar_try(mb, parity)) break;
      if (it >= W4_WAIT_LIMIT || s_dead) dead = true, s_dead = 1;
    }
    __syncwarp();
  };
  const int F = p.n_out;
  const int unit_rows = p.gated ? 8 : 16;   // of the weights, or of the gate's

  if (warp == W4_WARPS) {
    // ---- copies: a lane per box, gated two lanes ----
    if (!p.early) {
      if (mine > 0 && lane < W4_WARPS) {   // the first rows on their way to L2 while the block waits (a hint: no value is taken before the wait)
        const int row = (int)blockIdx.x * per_stage * unit_rows + lane;
        if (row < F) {
          const unsigned size = (unsigned)min(p.I / 2, 2048) & ~15u;
          asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p.w + (int64_t)row * (p.I / 2)), "r"(size) : "memory");
        }
      }
      pdl_wait();
      pdl_trigger();
    }
    bool waited = !p.early;
    const int box = p.gated ? lane & 15 : lane, half = p.gated ? lane >> 4 : 0;
    int q = 0, st = 0;
    unsigned phase = 0;   // of the copies
    for (int slice = 0; slice < p.slices; slice++)
      for (int i = 0; i < mine; i++) {
        const int set = (int)blockIdx.x + i * (int)gridDim.x;
        const int unit = set * per_stage + (box >> p.kw_log);
        for (int step = 0; step < steps; step++, q++) {
          if (!waited && q == p.stages) pdl_wait(), pdl_trigger(), waited = true;
          if (q >= p.stages) wait(empty + 8 * st, phase ^ 1);
          if (__any_sync(0xffffffffu, dead)) goto done;
          const int kb = step * kw + (box & (kw - 1)), col = (slice * p.boxes + kb) * (128 * SUB);   // bytes
          const bool on = box < W4_WARPS && unit < p.units && kb < p.boxes && col < p.I / 2;
          const int pieces = !on ? 0 : SUB == 1 || col + 128 >= p.I / 2 ? 1 : 2;
          const unsigned n = __reduce_add_sync(0xffffffffu, (unsigned)pieces);
          const unsigned mb = full + 8 * st;
          if (lane == 0) mbar_expect(mb, n * (p.gated ? W4_PIECE / 2 : W4_PIECE));
          __syncwarp();
#pragma unroll
          for (int sb = 0; sb < SUB; sb++)
            if (sb < pieces)
              tma_load2(base + st * W4_STAGE + box * W4_BOX + sb * W4_PIECE + half * (W4_PIECE / 2), &map, col + 128 * sb, unit * unit_rows + half * F, mb);
          if (++st == p.stages) st = 0, phase ^= 1;
        }
      }
  done:
    if (s_dead)   // what is under way has to land before the block ends
      for (int i = q < p.stages ? 0 : q - p.stages; i < q; i++)
        for (int it = 0; it < W4_WAIT_LIMIT && !mbar_try(full + 8 * (i % p.stages), (unsigned)(i / p.stages & 1)); it++) {}
    if (!waited) pdl_wait(), pdl_trigger();
    return;
  }

  if (warp == W4_WARPS + 1) {
    // ---- the sums of a unit's warps, and what becomes of them ----
    pdl_wait();
    pdl_trigger();
    int n_units = 0;
    for (int slice = 0; slice < p.slices; slice++)
      for (int i = 0; i < mine; i++, n_units++) {
        const int place = n_units % SUMS;
        wait(sums_full + 8 * place, (unsigned)(n_units / SUMS) & 1);
        const float* red = s_red + place * (W4_WARPS * 32 * 4 * NT);
        for (int j = 0; j < per_stage; j++) {
          const int unit = ((int)blockIdx.x + i * (int)gridDim.x) * per_stage + j;
          if (unit >= p.units) break;
#pragma unroll
          for (int n = 0; n < NT; n++) {
            float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
            for (int w = 0; w < kw; w++) {
              const float4 v = *reinterpret_cast<const float4*>(red + ((n * W4_WARPS + j * kw + w) * 32 + lane) * 4);
              y.x += v.x, y.y += v.y, y.z += v.z, y.w += v.w;
            }
            float4* part = reinterpret_cast<float4*>(p.partial) + ((int64_t)unit * 32 + lane) * NT + n;
            if (slice > 0) {
              const float4 v = *part;
              y.x += v.x, y.y += v.y, y.z += v.z, y.w += v.w;
            }
            if (slice + 1 < p.slices) {
              *part = y;
              continue;
            }
            *reinterpret_cast<float4*>(s_out + (n * 32 + lane) * 4) = y;
          }
          if (slice + 1 < p.slices) continue;
          __syncwarp();
          // row r, column c of the unit's sums
          auto sum_at = [&](int r, int c) { return s_out[(((c >> 3) * 32 + (r & 7) * 4 + ((c & 7) >> 1)) * 4) + (r >> 3) * 2 + (c & 1)]; };
          auto token = [&](int r, int t) {
            if (!WHOLE) return sum_at(r, t);
            float y = 0.0f;
#pragma unroll
            for (int d = W4_DIGITS - 1; d >= 0; d--) y += sum_at(r, d);   // the smallest first
            return y;
          };
          const int per_token = p.gated ? 8 : 16;
          for (int k = lane; k < per_token * p.T; k += 32) {
            const int t = k / per_token, r = k % per_token, o = unit * unit_rows + r;
            if (o >= F) continue;
            float y = token(r, t);
            if (p.gated) y = y / (1.0f + __expf(-y)) * token(r + 8, t);
            if (s_dead) y = NAN;
            p.out[(int64_t)t * F + o] = f2bf(y);
          }
          __syncwarp();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive1(sums_empty + 8 * place);
      }
    return;
  }

  // ---- products ----
  const int group = 1 << p.group_log, per_box = (256 * SUB) >> p.group_log, n_groups = p.I >> p.group_log;   // groups of a box, of a row
  // Scales and offsets of this warp's box, read two boxes ahead: groups t4, t4 + 4 .. of rows g and g + 8.  Behind the last row or group
  // the last one is read again: the outputs are dropped, x and the codes are zero there.
  struct Scales {
    uint16_t s[2][E], u[2][E];
  };
  const bool with_offsets = p.offsets != nullptr;
  int f_slice = 0, f_set = 0, f_step = 0, f_at = (warp & (kw - 1)) * per_box + t4, f_i0 = 0, f_i1 = 0;   // (numbers of scales fit 31 bits)
  auto fetch = [&](Scales& to) {
    if (f_slice == p.slices) return;
    if (f_step == 0) {
      const int unit = ((int)blockIdx.x + f_set * (int)gridDim.x) * per_stage + (warp >> p.kw_log);
      const int row0 = min(unit * unit_rows + g, F - 1), row1 = p.gated ? row0 + F : min(row0 + 8, F - 1);
      f_i0 = row0 * n_groups, f_i1 = row1 * n_groups;
    }
#pragma unroll
    for (int e = 0; e < E; e++)
      if (e == 0 || 4 * e < per_box) {
        const int a = min(f_at + 4 * e, n_groups - 1);
        to.s[0][e] = p.scales[f_i0 + a], to.s[1][e] = p.scales[f_i1 + a];
        if (with_offsets) to.u[0][e] = p.offsets[f_i0 + a], to.u[1][e] = p.offsets[f_i1 + a];
      }
    if (steps == 1 && p.slices == 1) {
      if (++f_set == mine) f_slice++;
      return;
    }
    if (++f_step == steps) {
      f_step = 0;
      if (++f_set == mine) f_set = 0, f_slice++;
    }
    f_at = (f_slice * p.boxes + f_step * kw + (warp & (kw - 1))) * per_box + t4;
  };
  if (!p.early) pdl_wait();   // (scales are weights too)
  Scales next = {}, after = {};
  fetch(next);
  fetch(after);
  if (p.early) pdl_wait();
  pdl_trigger();
  int st = 0, n_units = 0;
  unsigned phase = 0;
  uint32_t mask, magic;
  asm volatile("mov.b32 %0, 0x000f000f;\n\tmov.b32 %1, 0x43004300;" : "=r"(mask), "=r"(magic));
  const uint32_t bias = with_offsets ? 0x43004300u : 0x43084308u;   // 128, or 136
  unsigned d_lane[NT];   // this lane's column of x; of those that there are not a row of zeros
#pragma unroll
  for (int n = 0; n < NT; n++) d_lane[n] = smem_addr(s_dig) + min(g + 8 * n, PER * p.T) * p.pitch + 8 * BYTES * t4;
  for (int slice = 0; slice < p.slices; slice++) {
    // x of the slice: a warp takes 256 columns of a token, a lane eight; zeros behind the last column.
    const int first_col = slice * p.boxes * (256 * SUB), parts = p.boxes * SUB;
    if (slice > 0) asm volatile("bar.sync 1, 512;" ::: "memory");   // the last products with the digits before
    auto load_x = [&](int t, int part) -> uint4 {
      const int col = first_col + 256 * part + 8 * lane;
      return t < p.T && col < p.I ? *reinterpret_cast<const uint4*>(p.x + (int64_t)t * p.x_t + col) : make_uint4(0, 0, 0, 0);
    };
    int t = warp / parts, part = warp - t * parts, t_next, part_next;
    uint4 v = load_x(t, part), v_next;   // one turn ahead
    for (; t < p.T; t = t_next, part = part_next, v = v_next) {
      for (t_next = t, part_next = part + W4_WARPS; part_next >= parts; t_next++) part_next -= parts;
      v_next = load_x(t_next, part_next);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
      if constexpr (WHOLE) {
        uint32_t top = 0;   // the largest magnitude's bits
#pragma unroll
        for (int i = 0; i < 4; i++) top = max(top, max(w[i] & 0x7fffu, w[i] >> 16 & 0x7fffu));
        for (int off = group / 16; off > 0; off >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, off));
        const bool odd = top >= 0x7f80u;                           // an infinity or NaN: the token comes out as NaN
        const int k = max((int)(top >> 7), 7 * W4_DIGITS);         // largest value: [1, 2) 2^(k - 127), or less; the last digit's unit is 2^-126 at least
        float e = odd ? NAN : __uint_as_float((uint32_t)(k - 6) << 23);
        // A value is m 2^bit of the last digit's unit, m of 8 bits: two digits that follow one another, in their places of eight bytes.
        uint32_t lo[8], hi[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const uint32_t v = i & 1 ? w[i >> 1] >> 16 : w[i >> 1];
          const int exponent = (int)(v >> 7 & 255);
          uint32_t m = odd ? 0u : (v & 127) | (exponent ? 128u : 0u);
          int bit = max(exponent, 1) - k + 7 * W4_DIGITS - 8;
          m >>= min(max(-bit, 0), 31), bit = max(bit, 0);
          const int digit = bit * 37 >> 8;   // bit / 7, up to 48
          m <<= bit - 7 * digit;
          const int sign = v & 0x8000u ? -1 : 1;
          const uint32_t both = ((uint32_t)((int)(m & 127) * sign) & 255u) | ((uint32_t)((int)(m >> 7) * sign) & 255u) << 8;
          const uint64_t at = (uint64_t)both << (8 * digit);
          lo[i] = (uint32_t)at, hi[i] = (uint32_t)(at >> 32);
        }
#pragma unroll
        for (int half = 0; half < 2; half++) {   // the larger digits first
          const uint32_t(&x)[8] = half ? lo : hi;
          uint32_t even[4], uneven[4];           // [digit]: its bytes of the even columns, and of the others
          auto turn = [](uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t(&r)[4]) {
            const uint32_t ab0 = __byte_perm(a, b, 0x5140), ab1 = __byte_perm(a, b, 0x7362), cd0 = __byte_perm(c, d, 0x5140), cd1 = __byte_perm(c, d, 0x7362);
            r[3] = __byte_perm(ab0, cd0, 0x5410), r[2] = __byte_perm(ab0, cd0, 0x7632), r[1] = __byte_perm(ab1, cd1, 0x5410), r[0] = __byte_perm(ab1, cd1, 0x7632);
          };
          turn(x[0], x[2], x[4], x[6], even), turn(x[1], x[3], x[5], x[7], uneven);
#pragma unroll
          for (int j = 0; j < 4; j += 2) {   // two sums of 16 bits (at most 128 digits of 127) in a word
            uint32_t sums = 0;
#pragma unroll
            for (int i = 1; i >= 0; i--) sums = (sums << 16) + (uint32_t)__dp4a((int)even[j + i], 0x01010101, __dp4a((int)uneven[j + i], 0x01010101, 0));
            for (int off = group / 16; off > 0; off >>= 1) sums += __shfl_xor_sync(0xffffffffu, sums, off);
            const int sum0 = (int16_t)sums, sum1 = (int)(sums - (uint32_t)sum0) >> 16;
#pragma unroll
            for (int i = 0; i < 2; i++, e *= 0x1p-7f) {
              const int d = 4 * half + j + i, sum = i ? sum1 : sum0;
              *reinterpret_cast<uint2*>(s_dig + (PER * t + d) * p.pitch + 256 * part + 8 * lane) = make_uint2(even[j + i], uneven[j + i]);
              if ((lane & (group / 8 - 1)) == 0) {
                const int at = ((256 * part + 8 * lane) / group) * 8 * NT + PER * t + d;
                s_col[at] = {with_offsets ? W4_BIAS : W4_BIAS - 8u * (uint32_t)sum, e};
                if (with_offsets) s_x[at] = (float)sum * e;
              }
            }
          }
        }
      } else {
        // (0, 4), (1, 5), (2, 6), (3, 7): the order in which the codes' pairs come out of a word
        *reinterpret_cast<uint4*>(s_dig + t * p.pitch + 512 * part + 16 * lane) =
            make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x5410), __byte_perm(v.y, v.w, 0x7632));
        if (with_offsets) {
          float X = 0.0f;
#pragma unroll
          for (int e = 0; e < 4; e++) X += __uint_as_float(w[e] << 16) + __uint_as_float(w[e] & 0xffff0000u);
          for (int off = group / 16; off > 0; off >>= 1) X += __shfl_xor_sync(0xffffffffu, X, off);
          if ((lane & (group / 8 - 1)) == 0) s_x[((256 * part + 8 * lane) / group) * 8 * NT + t] = X;
        }
      }
    }
    if (PER * p.T < 8 * NT) {   // columns that there are not
      for (int i = tid; i < p.pitch / 8; i += 32 * W4_WARPS) *reinterpret_cast<uint2*>(s_dig + PER * p.T * p.pitch + 8 * i) = make_uint2(0, 0);
      if (with_offsets)
        for (int i = tid; i < p.groups_smem * (8 * NT - PER * p.T); i += 32 * W4_WARPS)
          s_x[i / (8 * NT - PER * p.T) * 8 * NT + PER * p.T + i % (8 * NT - PER * p.T)] = 0.0f;
    }
    asm volatile("bar.sync 1, 512;" ::: "memory");
    for (int i = 0; i < mine; i++) {
      const int unit = ((int)blockIdx.x + i * (int)gridDim.x) * per_stage + (warp >> p.kw_log);
      float total[NT][4] = {};
      for (int step = 0; step < steps; step++) {
        const Scales now = next;
        const int kb = step * kw + (warp & (kw - 1));
        next = after;
        fetch(after);
        wait(full + 8 * st, phase);
        if (kb < p.boxes && (slice * p.boxes + kb) * (256 * SUB) < p.I && unit < p.units) {   // warp-uniform
          const unsigned w_at = base + st * W4_STAGE + warp * W4_BOX + g * 128 + 4 * t4 + 16 * g, d_at = kb * (256 * SUB * BYTES);   // chunk 0 of row g, swizzled
          auto boxes = [&](auto log) {
            constexpr int CH = 1 << (decltype(log)::value - 5);   // steps of 32 columns in a group
#pragma unroll
            for (int c0 = 0; c0 < 8 * SUB; c0 += CH) {
              const int in_box = c0 / CH, from = (lane & 28) | (in_box & 3);
              uint32_t d[NT][4];
              float4 column[NT];   // whole numbers: of this lane's two columns, start and e
#pragma unroll
              for (int n = 0; n < NT; n++) {
                if constexpr (WHOLE) {
                  column[n] = *reinterpret_cast<const float4*>(s_col + (kb * per_box + in_box) * 8 * NT + 2 * t4 + 8 * n);
                  d[n][0] = d[n][2] = __float_as_uint(column[n].x), d[n][1] = d[n][3] = __float_as_uint(column[n].z);
                } else {
                  d[n][0] = d[n][1] = d[n][2] = d[n][3] = 0;
                }
              }
#pragma unroll
              for (int c = c0; c < c0 + CH; c++) {
                uint32_t w0, w1, b[NT][4];
                asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w0) : "r"((w_at ^ ((c & 7) << 4)) + (c >> 3) * W4_PIECE) : "memory");
                asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w1) : "r"((w_at ^ ((c & 7) << 4)) + (c >> 3) * W4_PIECE + 1024) : "memory");
                if constexpr (WHOLE) {
#pragma unroll
                  for (int n = 0; n < NT; n++)
                    asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(b[n][0]), "=r"(b[n][1]) : "r"(d_lane[n] + d_at + 32 * c) : "memory");
                  const uint32_t a0 = w0 & 0x0f0f0f0fu, a1 = w1 & 0x0f0f0f0fu, a2 = w0 >> 4 & 0x0f0f0f0fu, a3 = w1 >> 4 & 0x0f0f0f0fu;
#pragma unroll
                  for (int n = 0; n < NT; n++) mma_codes(d[n], a0, a1, a2, a3, b[n][0], b[n][1]);
                } else {
#pragma unroll
                  for (int n = 0; n < NT; n++)
                    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                                 : "=r"(b[n][0]), "=r"(b[n][1]), "=r"(b[n][2]), "=r"(b[n][3])
                                 : "r"(d_lane[n] + d_at + 64 * c)
                                 : "memory");
                  auto pair = [&](uint32_t w) { return less2(code_pair(w, mask, magic), bias); };
                  const uint32_t a0 = pair(w0), a1 = pair(w1), a2 = pair(w0 >> 4), a3 = pair(w1 >> 4), a4 = pair(w0 >> 8), a5 = pair(w1 >> 8), a6 = pair(w0 >> 12), a7 = pair(w1 >> 12);
#pragma unroll
                  for (int n = 0; n < NT; n++) {
                    mma_bf16(d[n], a0, a1, a2, a3, b[n][0], b[n][1]);
                    mma_bf16(d[n], a4, a5, a6, a7, b[n][2], b[n][3]);
                  }
                }
              }
              float sc[2];
#pragma unroll
              for (int r = 0; r < 2; r++) sc[r] = __uint_as_float(__shfl_sync(0xffffffffu, (uint32_t)now.s[r][in_box >> 2], from) << 16);
#pragma unroll
              for (int n = 0; n < NT; n++) {
                if constexpr (WHOLE) {
                  const float e0 = column[n].y, e1 = column[n].w, k0 = -12582912.0f * e0, k1 = -12582912.0f * e1;   // exact: e is a power of two
#pragma unroll
                  for (int e = 0; e < 4; e++) total[n][e] = fmaf(sc[e >> 1], fmaf(__uint_as_float(d[n][e]), e & 1 ? e1 : e0, e & 1 ? k1 : k0), total[n][e]);
                } else {
#pragma unroll
                  for (int e = 0; e < 4; e++) total[n][e] = fmaf(sc[e >> 1], __uint_as_float(d[n][e]), total[n][e]);
                }
              }
              if (with_offsets) {
                float u[2];
#pragma unroll
                for (int r = 0; r < 2; r++) u[r] = __uint_as_float(__shfl_sync(0xffffffffu, (uint32_t)now.u[r][in_box >> 2], from) << 16);
#pragma unroll
                for (int n = 0; n < NT; n++) {
                  const float2 sums = *reinterpret_cast<const float2*>(s_x + (kb * per_box + in_box) * 8 * NT + 2 * t4 + 8 * n);
#pragma unroll
                  for (int e = 0; e < 4; e++) total[n][e] = fmaf(u[e >> 1], e & 1 ? sums.y : sums.x, total[n][e]);
                }
              }
            }
          };
          if (p.group_log == 7) boxes(std::integral_constant<int, 7>());
          else if (p.group_log == 6) boxes(std::integral_constant<int, 6>());
          else boxes(std::integral_constant<int, 5>());
        }
        __syncwarp();
        if (lane == 0) mbar_arrive1(empty + 8 * st);
        if (++st == p.stages) st = 0, phase ^= 1;
      }
      // ---- this warp's sums of the unit ----
      const int place = n_units % SUMS;
      if (n_units >= SUMS) wait(sums_empty + 8 * place, (unsigned)(n_units / SUMS - 1) & 1);
      float* red = s_red + place * (W4_WARPS * 32 * 4 * NT);
#pragma unroll
      for (int n = 0; n < NT; n++) *reinterpret_cast<float4*>(red + ((n * W4_WARPS + warp) * 32 + lane) * 4) = make_float4(total[n][0], total[n][1], total[n][2], total[n][3]);
      __syncwarp();
      if (lane == 0) mbar_arrive1(sums_full + 8 * place);
      n_units++;
    }
  }
}

// How x and the rows are laid out for a product.
struct W4Plan {
  bool whole;
  int tiles, sub, stages, units, boxes, kw_log, slices, pitch, groups_smem, smem, sets;
};
W4Plan w4_plan(int64_t n_out, int64_t I, int64_t T, int group_log, bool gated, bool offsets, bool whole, int sub) {
  W4Plan r = {};
  const int columns = (int)(whole ? W4_DIGITS * T : T), NT = (columns + 7) / 8, bytes = whole ? 1 : 2;
  r.whole = whole, r.tiles = NT, r.sub = sub;
  r.units = (int)(gated ? (n_out + 7) / 8 : (n_out + 15) / 16);
  const int all = (int)((I + 256 * sub - 1) / (256 * sub)), stage = W4_WARPS * sub * W4_PIECE, fixed = 1024 + 2 * stage + w4_sums(NT) * W4_WARPS * 32 * 16 * NT + 512 * NT;
  for (r.slices = 1;; r.slices++) {
    r.boxes = (all + r.slices - 1) / r.slices;
    if (r.slices > 1 && r.boxes > W4_WARPS) r.boxes = (r.boxes + W4_WARPS - 1) / W4_WARPS * W4_WARPS;   // whole stages, but for the last
    r.pitch = r.boxes * 256 * sub * bytes + 32 * bytes;   // (four columns' 32 bytes, or two columns' 64, fill the banks)
    r.groups_smem = r.boxes * ((256 * sub) >> group_log);
    r.smem = fixed + r.groups_smem * 8 * NT * ((whole ? 8 : 0) + (offsets ? 4 : 0)) + (columns + (columns % 8 != 0)) * r.pitch;
    if (r.smem <= W4_SMEM || r.boxes == 1) break;
  }
  r.slices = (all + r.boxes - 1) / r.boxes;
  for (r.stages = 2; r.stages < W4_STAGES_MAX && r.smem + stage <= W4_SMEM; r.stages++) r.smem += stage;
  while ((1 << r.kw_log) < r.boxes && (1 << r.kw_log) < W4_WARPS) r.kw_log++;
  r.sets = (r.units + (W4_WARPS >> r.kw_log) - 1) / (W4_WARPS >> r.kw_log);
  return r;
}
// Boxes of 512 columns, which spread what a box costs besides its products, from eight stages per SM on; for one token in whole numbers, where all of its
// digits fit at once.  Nine tokens and more, whose sums take two columns of eight and whose x then fits in fewer pieces, have boxes of 256.  B200, us, caches cold, events around a call, groups of 128 | of 64 with offsets.  One token, whole numbers, bf16 in boxes of 512,
// of 256:  24576 x 4096 (5 stages per SM) 25.6, 25.6, 26.7 | gated 32.7, 30.8, 30.7;  36000 x 4096 (8) 30.8, 31.7, 34.8 | 38.9, 38.9, 39.9;  151936 x 4096 (32)
// 80.8, 97.2, 112 | 109, 119, 128;  19000 x 12288 in two pieces 56.4, 51.3, 49.1.  Bf16 in boxes of 512, of 256:  six tokens, 24576 x 4096 gated 37.0, 34.9,
// 36000 x 4096 42.9, 43.1, 64000 x 4096 gated 65.5, 67.6;  eight tokens, 151936 x 4096 104, 119, 19000 x 12288 64, 72, 19000 x 16384 82, 78;  nine, 151936 x 4096 233, 154;  sixteen, the same 339, 236, 24576 x 4096 78, 55,
// twelve, 152000 x 768 111, 113.
W4Plan w4_plan(int64_t n_out, int64_t I, int64_t T, int group_log, bool gated, bool offsets) {
  for (const bool whole : {T == 1, false}) {
    if (T > 8) break;
    const W4Plan two = w4_plan(n_out, I, T, group_log, gated, offsets, whole, 2);
    const int64_t stages = (int64_t)two.sets * ((two.boxes + (1 << two.kw_log) - 1) >> two.kw_log);
    if (stages >= W4_LONG * (int64_t)sm_count() && !(whole && two.slices > 1)) return two;
  }
  return w4_plan(n_out, I, T, group_log, gated, offsets, false, 1);
}

}  // namespace
}  // namespace pk

using namespace pk;

extern "C" int64_t pk_gemv_w4_workspace_bytes(int64_t T, int64_t O, int64_t I, int64_t group, int gated) {
  if (T < 1 || T > 16 || O < 1 || O >= (1LL << 30) || I < 32 || I > 32768 || (group != 32 && group != 64 && group != 128)) return 0;
  // (the larger of what is needed with offsets and without)
  int64_t most = 0;
  for (const bool offsets : {false, true}) {
    const W4Plan plan = w4_plan(gated ? O / 2 : O, I, T, group == 128 ? 7 : group == 64 ? 6 : 5, gated != 0, offsets);
    if (plan.slices > 1) most = (int64_t)plan.units * 32 * 16 * plan.tiles;
  }
  return most;
}

extern "C" int pk_gemv_w4(const pk_tensor* weight, const pk_tensor* scales, const pk_tensor* offsets, const pk_tensor* x, const pk_tensor* out,
                          int gated, void* workspace, int64_t workspace_bytes, void* stream) {
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
  PK_REQUIRE(O * groups < (1LL << 31), "sizes out of range");
  PK_REQUIRE(!gated || O % 2 == 0, "a gated product takes an even number of rows");
  PK_REQUIRE(is_contig(out) && out->shape[0] == T && out->shape[1] == (gated ? O / 2 : O), "out must be contiguous bf16 [T,O] (O/2 when gated)");
  PK_REQUIRE(aligned16(weight->data) && aligned16(x->data), "weight and x must be 16-byte aligned");
  if (T == 0) return PK_OK;
  const int n_out = (int)(gated ? O / 2 : O), group_log = group == 128 ? 7 : group == 64 ? 6 : 5;
  const W4Plan plan = w4_plan(n_out, I, T, group_log, gated != 0, offsets != nullptr);
  if (plan.slices > 1 && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255) || workspace_bytes < pk_gemv_w4_workspace_bytes(T, O, I, group, gated)))
    return fail(PK_ERR_WORKSPACE, "gemv_w4: workspace missing, misaligned or too small");
  CUtensorMap map;
  const auto encode = tensor_map_encoder();
  const cuuint64_t dims[2] = {(cuuint64_t)(I / 2), (cuuint64_t)O}, strides[1] = {(cuuint64_t)(I / 2)};
  const cuuint32_t box[2] = {128, gated ? 8u : 16u}, ones[2] = {1, 1};
  if (!encode || encode(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, weight->data, dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return fail(PK_ERR_CUDA, "gemv_w4: the driver made no tensor map of the weights");
  W4Params p = {};
  p.w = (const uint8_t*)weight->data, p.scales = (const uint16_t*)scales->data, p.offsets = offsets ? (const uint16_t*)offsets->data : nullptr;
  p.x = (const uint16_t*)x->data, p.x_t = x->stride[0], p.out = (uint16_t*)out->data;
  p.n_out = n_out, p.I = (int)I, p.T = (int)T, p.group_log = group_log, p.gated = gated != 0;
  p.units = plan.units, p.boxes = plan.boxes, p.kw_log = plan.kw_log, p.stages = plan.stages, p.slices = plan.slices, p.pitch = plan.pitch, p.groups_smem = plan.groups_smem;
  p.partial = (float*)workspace, p.early = pdl_early();
  const unsigned grid = (unsigned)(plan.sets < sm_count() ? plan.sets : sm_count());
  StageTimer timer(ST_GEMV, (cudaStream_t)stream);
  auto launch = [&](auto whole, auto nt, auto sub) -> int {
    constexpr bool WHOLE = decltype(whole)::value;
    constexpr int NT = decltype(nt)::value, SUB = decltype(sub)::value;
    static PerDevice opted;
    if (const unsigned long long bit = first_on_device(opted)) {
      if (cudaFuncSetAttribute(gemv_w4_kernel<WHOLE, NT, SUB>, cudaFuncAttributeMaxDynamicSharedMemorySize, W4_SMEM) != cudaSuccess)
        return fail(PK_ERR_CUDA, "gemv_w4: %s", cudaGetErrorString(cudaGetLastError()));
      mark_on_device(opted, bit);
    }
    launch_chain(gemv_w4_kernel<WHOLE, NT, SUB>, dim3(grid), dim3(W4_THREADS), (size_t)plan.smem, (cudaStream_t)stream, map, p);
    return PK_OK;
  };
  using One = std::integral_constant<int, 1>;
  using Two = std::integral_constant<int, 2>;
  using Bf16 = std::false_type;
  const int rc = plan.whole ? launch(std::true_type(), One(), Two())
                 : plan.tiles == 2 ? launch(Bf16(), Two(), One())
                 : plan.sub == 2   ? launch(Bf16(), One(), Two())
                                   : launch(Bf16(), One(), One());
  if (rc) return rc;
  return check_launch("gemv_w4");
}
