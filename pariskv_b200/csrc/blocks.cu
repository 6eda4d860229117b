// Block bounds of the keys of a cache, and the selection of blocks by them.
//   bounds[j] = (lo, hi): smallest and largest value per channel over the rows of block j
//   score_j   = sum_d sum_g max(q_gd lo_jd, q_gd hi_jd), no less than the sum over the group's query heads g of q_g.k for any key k of the
//               block;  with P_d = sum_g max(q_gd, 0) and N_d = sum_g min(q_gd, 0) it is sum_d P_d hi_jd + N_d lo_jd: one pass over the
//               bounds whatever the number of query heads.
// The choice is that of sums in 64 bits, rounded once to 32: it does not depend on their order.
#include <type_traits>

#include "attend.cuh"
#include "tma.cuh"

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
  int64_t o_b, o_h, o_j, nb, cap;   // cap: rows of the cache, in nb blocks
  const int32_t* lengths;
  int T, H, G, n, block, sink, local;
  uint32_t* keys;      // [rows][nb] ordered keys of the scores
  float* limits;       // [rows][warps of the score kernel on a row]
  int32_t* ids;        // [rows][n]
};

// Keys order as the scores do.  NaN is above all numbers, what is always taken above that; 0: a block that is not seen.
constexpr uint32_t FORCED = 0xffffffffu, NOT_A_NUMBER = 0xfffffffeu;

// Blocks that row (b, t) sees.
__device__ __forceinline__ int visible_blocks(const SelectParams& p, int64_t b, int t) {
  const int64_t pos = min((int64_t)p.lengths[b], p.cap) - p.T + t;
  return pos < 0 ? 0 : (int)(pos / p.block) + 1;
}

// Sums of eight values over the lanes of a warp; lane L gets that of value L / 4.
__device__ __forceinline__ float warp_sums8(float (&v)[8], int lane) {
#pragma unroll
  for (int n = 4, off = 16; n >= 1; n /= 2, off /= 2) {
    const bool up = lane & off;
#pragma unroll
    for (int i = 0; i < n; i++) {
      const float keep = up ? v[i + n] : v[i], give = up ? v[i] : v[i + n];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, give, off);
    }
  }
  v[0] += __shfl_xor_sync(0xffffffffu, v[0], 2);
  v[0] += __shfl_xor_sync(0xffffffffu, v[0], 1);
  return v[0];
}
// P (lanes 16 .. 31) or N (0 .. 15) of eight channels of token t: sums over the group's heads, four loads in flight.
template <class F>
__device__ __forceinline__ void query_sums(const SelectParams& p, int64_t b, int t, int h, int lane, F (&c)[8]) {
  const uint16_t* q = p.q + b * p.q_b + (int64_t)t * p.q_t + (int64_t)h * p.G * p.q_h + 8 * (lane & 15);
#pragma unroll
  for (int e = 0; e < 8; e++) c[e] = 0;
  for (int g0 = 0; g0 < p.G; g0 += 4) {
    uint4 x[4];
#pragma unroll
    for (int g = 0; g < 4; g++) x[g] = g0 + g < p.G ? *reinterpret_cast<const uint4*>(q + (g0 + g) * p.q_h) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int g = 0; g < 4; g++) {
      const uint32_t w[4] = {x[g].x, x[g].y, x[g].z, x[g].w};
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const float v = __uint_as_float(e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16);
        if (lane >= 16 ? !(v < 0.0f) : v < 0.0f) c[e] += (F)v;
      }
    }
  }
}

// Scores in 32 bits, and a bound A of every sum of absolute values: A = sum_d P_d max |hi_d| + |N_d| max |lo_d| over the warp's blocks.  A score is off
// by at most G + 13 roundings of 2^-24 A (P or N, eight products in a row, five additions of the lanes' sums): where the choice hangs on less
// than that, block_pick_kernel takes the 64-bit scores.  Products below 2^-100 count as that much in A, which leaves room for what 32 bits lose where they hold
// numbers by fewer digits: A is zero only where every product is.
// A warp of its own brings 32 blocks of keys at a time, 16 KB, into a ring of four stages; each of four warps takes eight of them for TT tokens: lanes
// 0 .. 15 hold eight channels of lo and N each, the others of hi and P.  Bounded by the bounds' bytes where there are many, otherwise by
// latency.  With the choice, us a call in a replayed graph, bounds in HBM (in L2): 8192 blocks of 8 heads for four tokens 23.0 (21.0), for one 16.3 (14.2),
// 512 blocks 5.9 (5.9), 128 heads x 400 blocks 11.5 (10.0).  Call after call, which adds the launches: by loads to registers two groups
// ahead | by the ring 29 | 28, 21 | 18, 8.3 | 7.7;  copies of one block each, which bounds with gaps need, cost more the more of them there are: 128 heads x 400
// blocks 14.5, in copies of 512 bytes 16.5.  (64-bit sums throughout: four tokens 46 us for the scores alone; the conversions to 64 bits, 8
// a clock and SM, take longer than the bytes.)
constexpr int SCORE_BLOCKS = 32, SCORE_STAGE = 512 * SCORE_BLOCKS, SCORE_STAGES = 4, SCORE_THREADS = 160, SCORE_CTAS = 3;   // blocks per SM, by the registers
constexpr int SCORE_WAIT_LIMIT = 100000;   // tries; one waits up to 10 us by itself
template <int TT>
__global__ void __launch_bounds__(SCORE_THREADS, SCORE_CTAS) block_score_kernel(SelectParams p) {
  extern __shared__ __align__(128) unsigned char ring[];
  __shared__ __align__(8) unsigned long long bars[2 * SCORE_STAGES];
  __shared__ volatile int s_dead;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, h = blockIdx.y % p.H, t0 = blockIdx.y / p.H * TT;
  const unsigned full = smem_addr(bars), empty = full + 8 * SCORE_STAGES;
  if (threadIdx.x == 0) {
    for (int i = 0; i < SCORE_STAGES; i++) mbar_init(full + 8 * i, 1), mbar_init(empty + 8 * i, 4);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    s_dead = 0;
  }
  __syncthreads();
  pdl_wait();
  pdl_trigger();
  const int64_t b = blockIdx.z;
  int seen[TT], most = 0;
#pragma unroll
  for (int i = 0; i < TT; i++) seen[i] = t0 + i < p.T ? visible_blocks(p, b, t0 + i) : 0, most = max(most, seen[i]);
  const int steps = (most + SCORE_BLOCKS - 1) / SCORE_BLOCKS;
  bool dead = false;   // a wait has run out: no more waiting; the limits become NaN, and the choice is made of 64-bit sums
  auto wait = [&](unsigned mb, unsigned parity) {
    for (int it = 0; !dead; it++) {
      if (mbar_try(mb, parity)) break;
      if (it >= SCORE_WAIT_LIMIT || s_dead) dead = true, s_dead = 1;
    }
    __syncwarp();
  };
  if (warp == 4) {
    const uint16_t* bounds = p.bounds + b * p.o_b + h * p.o_h;
    int q = 0;
    for (int step = blockIdx.x; step < steps; step += gridDim.x, q++) {
      const int st = q % SCORE_STAGES, n = min(SCORE_BLOCKS, most - SCORE_BLOCKS * step);
      if (q >= SCORE_STAGES) wait(empty + 8 * st, (unsigned)(q / SCORE_STAGES - 1) & 1);
      if (__any_sync(0xffffffffu, dead)) break;
      if (lane == 0) mbar_expect(full + 8 * st, 512 * n);
      __syncwarp();
      const int per = p.o_j == 256 ? 8 : 1, first = per * lane;   // blocks of a copy
      if (first < n)
        bulk_load(smem_addr(ring) + st * SCORE_STAGE + 512 * first, bounds + (int64_t)(SCORE_BLOCKS * step + first) * p.o_j, 512 * min(per, n - first), full + 8 * st);
    }
    if (s_dead)   // what is under way has to land before the block ends
      for (int i = q < SCORE_STAGES ? 0 : q - SCORE_STAGES; i < q; i++)
        for (int it = 0; it < SCORE_WAIT_LIMIT && !mbar_try(full + 8 * (i % SCORE_STAGES), (unsigned)(i / SCORE_STAGES & 1)); it++) {}
    return;
  }
  const int warps = (int)gridDim.x * 4, self = (int)blockIdx.x * 4 + warp;
  // P and N of the block's tokens, a thread per channel
  __shared__ __align__(16) float s_sums[TT][2][128];
  {
    const int d = threadIdx.x;
    float up[TT], down[TT];
#pragma unroll
    for (int i = 0; i < TT; i++) up[i] = down[i] = 0.0f;
    const uint16_t* q = p.q + b * p.q_b + (int64_t)h * p.G * p.q_h + d;
    for (int g0 = 0; g0 < p.G; g0 += 4) {
      float v[TT][4];
#pragma unroll
      for (int i = 0; i < TT; i++)
#pragma unroll
        for (int g = 0; g < 4; g++) v[i][g] = g0 + g < p.G ? bf2f(q[(int64_t)min(t0 + i, p.T - 1) * p.q_t + (g0 + g) * p.q_h]) : 0.0f;
#pragma unroll
      for (int i = 0; i < TT; i++)
#pragma unroll
        for (int g = 0; g < 4; g++) {
          if (v[i][g] < 0.0f) down[i] += v[i][g];
          else up[i] += v[i][g];
        }
    }
#pragma unroll
    for (int i = 0; i < TT; i++) s_sums[i][0][d] = down[i], s_sums[i][1][d] = up[i];
  }
  asm volatile("bar.sync 1, 128;" ::: "memory");
  float c[TT][8];   // P or N of this lane's channels
#pragma unroll
  for (int i = 0; i < TT; i++)
#pragma unroll
    for (int e = 0; e < 8; e += 4) *reinterpret_cast<float4*>(&c[i][e]) = *reinterpret_cast<const float4*>(&s_sums[i][lane >> 4][8 * (lane & 15) + e]);
  __nv_bfloat162 top[4];   // largest magnitudes of this lane's channels
#pragma unroll
  for (int e = 0; e < 4; e++) top[e] = __nv_bfloat162(__ushort_as_bfloat16(0), __ushort_as_bfloat16(0));
  int q = 0;
  for (int step = blockIdx.x; step < steps; step += gridDim.x, q++) {
    const int st = q % SCORE_STAGES, first = SCORE_BLOCKS * step + 8 * warp;
    wait(full + 8 * st, (unsigned)(q / SCORE_STAGES) & 1);
    const uint4* from = reinterpret_cast<const uint4*>(ring + st * SCORE_STAGE + 4096 * warp) + lane;
    float sum[TT][8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const uint4 x = first + i < most ? from[32 * i] : make_uint4(0, 0, 0, 0);
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
      float v[8];
#pragma unroll
      for (int e = 0; e < 4; e++) {
        v[2 * e] = __uint_as_float(w[e] << 16), v[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
        top[e] = __hmax2_nan(top[e], __habs2(*reinterpret_cast<const __nv_bfloat162*>(&w[e])));
      }
#pragma unroll
      for (int k = 0; k < TT; k++) {
        float s = c[k][0] * v[0];
#pragma unroll
        for (int e = 1; e < 8; e++) s = fmaf(c[k][e], v[e], s);
        sum[k][i] = s;
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive1(empty + 8 * st);
#pragma unroll
    for (int k = 0; k < TT; k++) {
      const float f = warp_sums8(sum[k], lane) + 0.0f;   // (one zero)
      const int j = first + (lane >> 2);
      if ((lane & 3) == 0 && j < seen[k])
        p.keys[((b * p.T + t0 + k) * p.H + h) * p.nb + j] = j < p.sink || j >= seen[k] - p.local ? FORCED : f != f ? NOT_A_NUMBER : ord_key(f);
    }
  }
#pragma unroll
  for (int k = 0; k < TT; k++) {
    float A = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; e++) {   // (infinite bounds: inf or NaN)
      const float x = fabsf(c[k][e]), y = e & 1 ? __high2float(top[e >> 1]) : __low2float(top[e >> 1]), a = x * y;
      A += a < 0x1p-100f && x != 0.0f && y != 0.0f ? 0x1p-100f : a;
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) A += __shfl_xor_sync(0xffffffffu, A, off);
    if (lane == 0 && t0 + k < p.T) p.limits[((b * p.T + t0 + k) * p.H + h) * warps + self] = dead ? NAN : A;
  }
}

// A block per row, a thread holds KPT of its keys.  The keys between the lowest and the highest are counted in 1024 bins of equal width, the bin of the n-th
// largest is cut again until it is taken whole or holds one value (of which the lowest positions are taken); usually one or two rounds.
// What is taken is listed and ranked by position.  Where the lowest score taken and the highest one left lie closer than the rounding of the
// scores, those in question are summed again in 64 bits and chosen from once more; then, and where a value is taken in part or more than
// PICK_LIST are, the chosen ones come out in order, every warp those of its part of the row.  Latency: a barrier and a pass over registers a
// step.  (Keys in shared memory, 512 threads, every row written in order: 32 rows of 8192 keys 10 us, of which 3.5 for the order.)
constexpr int PICK_THREADS = 1024, PICK_WARPS = PICK_THREADS / 32, PICK_BINS = 1024, PICK_LIST = 1024;
template <int KPT>
__global__ void __launch_bounds__(PICK_THREADS) block_pick_kernel(SelectParams p, int warps) {
  __shared__ unsigned s_bins[2][PICK_BINS], s_a[PICK_WARPS], s_b[PICK_WARPS], s_c[PICK_WARPS], s_d[PICK_WARPS], s_found[3], s_n;
  __shared__ int s_list[PICK_LIST];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t row = blockIdx.x, t = row / p.H % p.T, b = row / p.H / p.T;
  const int h = (int)(row % p.H);
  s_bins[0][tid] = 0, s_bins[1][tid] = 0;
  if (tid == 0) s_n = 0;
  pdl_wait();
  pdl_trigger();
  const int seen = visible_blocks(p, b, (int)t);
  uint32_t* stored = p.keys + row * p.nb;
  int32_t* ids = p.ids + row * p.n;
  for (int i = min(p.n, seen) + tid; i < p.n; i += PICK_THREADS) ids[i] = -1;
  if (seen <= p.n) {   // all of them
    for (int i = tid; i < seen; i += PICK_THREADS) ids[i] = i;
    return;
  }
  // KPT = 0: more keys than fit, read from global memory in every pass
  uint32_t kept[KPT > 0 ? KPT : 1];
  if (KPT > 0)
#pragma unroll
    for (int i = 0; i < KPT; i++) kept[i] = i * PICK_THREADS + tid < seen ? stored[i * PICK_THREADS + tid] : 0u;
  // f(position, key) for this thread's keys; 0 is the key of what is not chosen from
  auto each = [&](auto&& f) {
    if (KPT > 0) {
#pragma unroll
      for (int i = 0; i < KPT; i++)
        if (i * PICK_THREADS + tid < seen) f(i * PICK_THREADS + tid, kept[i]);
    } else {
      for (int j = tid; j < seen; j += PICK_THREADS) f(j, stored[j]);
    }
  };
  auto value = [](uint32_t k) { return __uint_as_float((k & 0x80000000u) ? (k ^ 0x80000000u) : ~k); };
  // lowest, two highest and a sum over the block, to every thread
  auto range = [&](uint32_t& lo, uint32_t& hi, uint32_t& hi2, unsigned& n) {
    lo = __reduce_min_sync(0xffffffffu, lo), hi = __reduce_max_sync(0xffffffffu, hi), hi2 = __reduce_max_sync(0xffffffffu, hi2), n = __reduce_add_sync(0xffffffffu, n);
    __syncthreads();
    if (lane == 0) s_a[warp] = lo, s_b[warp] = hi, s_c[warp] = n, s_d[warp] = hi2;
    __syncthreads();
    lo = __reduce_min_sync(0xffffffffu, s_a[lane]), hi = __reduce_max_sync(0xffffffffu, s_b[lane]);
    n = __reduce_add_sync(0xffffffffu, s_c[lane]), hi2 = __reduce_max_sync(0xffffffffu, s_d[lane]);
  };
  uint32_t lo = 0xffffffffu, hi = 0, limit = 0;   // extremes of the keys that are not FORCED; the largest limit's bits
  unsigned forced = 0;
  for (int i = tid; i < warps; i += PICK_THREADS) {
    const float a = p.limits[row * warps + i];
    limit = max(limit, a <= 3.0e38f ? __float_as_uint(a) : 0x7f800000u);
  }
  each([&](int, uint32_t k) {
    if (k == FORCED) forced++;
    else lo = min(lo, k), hi = max(hi, k);
  });
  range(lo, hi, limit, forced);
  const float A = __uint_as_float(limit);
  unsigned want = 0;
  int round = 0;
  // Narrows [lo, hi] to keys of which `want` are taken (all of them, or equal ones), those above hi being taken as well.
  auto narrow = [&]() {
    want = (unsigned)p.n - forced;   // (more blocks than are taken are seen, and the forced ones are at most n: there are others)
    unsigned in_range = 0xffffffffu;
    for (; want > 0 && want != in_range && lo != hi; round++) {
      unsigned* bins = s_bins[round & 1];
      const int shift = max(0, 22 - __clz(hi - lo));   // (hi - lo) >> shift < 1024
      each([&](int, uint32_t k) {
        if (k >= lo && k <= hi && k != FORCED) atomicAdd(&bins[(k - lo) >> shift], 1u);
      });
      __syncthreads();
      const unsigned c = bins[PICK_BINS - 1 - tid];   // from the highest down
      unsigned sum = c;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const unsigned o = __shfl_up_sync(0xffffffffu, sum, off);
        if (lane >= off) sum += o;
      }
      if (lane == 31) s_a[warp] = sum;
      __syncthreads();
      bins[PICK_BINS - 1 - tid] = 0;   // for the round after the next
      const unsigned before = __reduce_add_sync(0xffffffffu, lane < warp ? s_a[lane] : 0u) + sum - c;
      if (before < want && before + c >= want) s_found[0] = PICK_BINS - 1 - tid, s_found[1] = before, s_found[2] = c;
      __syncthreads();
      lo += s_found[0] << shift;
      hi = lo + min(hi - lo, (1u << shift) - 1);   // (NaN's bin ends behind the last 32-bit number)
      want -= s_found[1], in_range = s_found[2];
    }
    return lo == hi && want != in_range;   // taken in part
  };
  bool part = narrow(), listed = p.n <= PICK_LIST;
  {
    // the lowest key taken and the highest one left, and the list of what is taken
    uint32_t low = 0xffffffffu, high = 0, high2 = 0;
    unsigned none = 0;
    const bool only_forced = forced == (unsigned)p.n;
    each([&](int j, uint32_t k) {
      const bool taken = k == FORCED || (!only_forced && k >= lo);
      if (k != FORCED) {
        if (taken) low = min(low, k);
        if (!taken || part) high = max(high, k <= hi || only_forced ? k : 0u);
      }
      if (taken && listed && !part) {
        const unsigned at = atomicAdd(&s_n, 1u);
        if (at < PICK_LIST) s_list[at] = j;
      }
    });
    range(low, high, high2, none);
    const float margin = 2.5f * (float)(p.G + 14) * 0x1p-24f * A;   // of each of two scores G + 13 roundings and one more to 32 bits, with room
    const bool odd = !(A < 3.0e38f);
    const bool settled = only_forced || (!odd && (part ? A == 0.0f : value(low) - value(high) > margin));
    if (settled && listed && !part) {
      for (int i = tid; i < p.n; i += PICK_THREADS) {
        const int j = s_list[i];
        int rank = 0;
        for (int o = 0; o < p.n; o++) rank += s_list[o] < j;
        ids[rank] = j;
      }
      return;
    }
    if (!settled) {
      const float upper = value(high) + margin, lower = value(low) - margin;
      // those in question, a warp each; the others are settled
      double c[8];
      query_sums(p, b, (int)t, h, lane, c);
      const uint16_t* bounds = p.bounds + b * p.o_b + h * p.o_h + 8 * lane;
      lo = 0xffffffffu, hi = 0, forced = 0;
      auto again = [&](int j, uint32_t k) -> uint32_t {   // by a whole warp: j of its lanes
        bool open = false;
        if (j < seen && k != FORCED && k != 0) {
          const float s = value(k);
          open = odd || (s <= upper && s >= lower);
          if (!open) k = s > upper ? FORCED : 0u;
        }
        for (unsigned left = __ballot_sync(0xffffffffu, open); left; left &= left - 1) {
          const int i = __ffs(left) - 1;
          const uint4 x = *reinterpret_cast<const uint4*>(bounds + (int64_t)(j - lane + i) * p.o_j);
          const uint32_t w[4] = {x.x, x.y, x.z, x.w};
          double s = 0.0;
#pragma unroll
          for (int e = 0; e < 8; e++)   // (no products of a zero with an infinite bound)
            if (!(c[e] == 0.0)) s = fma(c[e], (double)__uint_as_float(e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16), s);
#pragma unroll
          for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
          const float f = (float)s + 0.0f;
          if (lane == i) k = f != f ? NOT_A_NUMBER : ord_key(f);
        }
        if (j < seen) {
          if (k == FORCED) forced++;
          else lo = min(lo, k), hi = max(hi, k);
        }
        return k;
      };
      if (KPT > 0) {
#pragma unroll
        for (int i = 0; i < KPT; i++) kept[i] = again(i * PICK_THREADS + tid, kept[i]);
      } else {
        for (int j0 = 32 * warp; j0 < seen; j0 += PICK_THREADS) {
          const uint32_t k = again(j0 + lane, j0 + lane < seen ? stored[j0 + lane] : 0u);
          if (j0 + lane < seen) stored[j0 + lane] = k;
        }
      }
      uint32_t none2 = 0;
      range(lo, hi, none2, forced);
      narrow();
    }
  }
  // In order: above hi, or FORCED: taken; in [lo, hi]: the first `want`.
  auto is_above = [&](uint32_t k) { return k == FORCED || (want > 0 && k > hi); };
  if (KPT > 0)
#pragma unroll
    for (int i = 0; i < KPT; i++)
      if (i * PICK_THREADS + tid < seen) stored[i * PICK_THREADS + tid] = kept[i];
  __syncthreads();
  const int per = ((seen + PICK_WARPS - 1) / PICK_WARPS + 31) / 32 * 32, j0 = min(seen, warp * per), j1 = min(seen, j0 + per);
  unsigned above = 0, inside = 0;
  for (int j = j0 + lane; j < j1; j += 32) {
    const uint32_t k = stored[j];
    if (is_above(k)) above++;
    else if (k >= lo && want > 0) inside++;
  }
  above = __reduce_add_sync(0xffffffffu, above), inside = __reduce_add_sync(0xffffffffu, inside);
  if (lane == 0) s_a[warp] = above, s_b[warp] = inside;
  __syncthreads();
  unsigned n_above = __reduce_add_sync(0xffffffffu, lane < warp ? s_a[lane] : 0u), n_inside = __reduce_add_sync(0xffffffffu, lane < warp ? s_b[lane] : 0u);
  for (int j = j0; j < j1; j += 32) {
    const uint32_t k = j + lane < j1 ? stored[j + lane] : 0;
    const bool a = j + lane < j1 && is_above(k), i = j + lane < j1 && !a && want > 0 && k >= lo;
    const unsigned ab = __ballot_sync(0xffffffffu, a), ib = __ballot_sync(0xffffffffu, i), below = (1u << lane) - 1;
    const unsigned i_at = n_inside + __popc(ib & below), at = n_above + __popc(ab & below) + min(i_at, want);
    if (a || (i && i_at < want)) ids[at] = j + lane;
    n_above += __popc(ab), n_inside += __popc(ib);
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
  for (int i = 0; i < 3; i++) PK_REQUIRE(bounds->shape[i] <= 1 || bounds->stride[i] > 0, "bounds are written: heads or blocks of them must not share memory");
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

extern "C" int64_t pk_select_blocks_workspace_bytes(int64_t bs, int64_t T, int64_t H, int64_t n_blocks) {
  return bs * T * H * (n_blocks + 4 * ((n_blocks + 31) / 32)) * 4 + 256;   // keys, and a limit for every warp
}

extern "C" int pk_select_blocks(const pk_tensor* queries, const pk_tensor* bounds, const pk_tensor* lengths, int64_t block, int64_t sink_blocks,
                                int64_t local_blocks, const pk_tensor* blocks, void* workspace, int64_t workspace_bytes, void* stream) {
  return pk_select_blocks_ex(queries, bounds, lengths, block, -1, sink_blocks, local_blocks, blocks, workspace, workspace_bytes, stream);
}

extern "C" int pk_select_blocks_ex(const pk_tensor* queries, const pk_tensor* bounds, const pk_tensor* lengths, int64_t block, int64_t cap,
                                   int64_t sink_blocks, int64_t local_blocks, const pk_tensor* blocks, void* workspace,
                                   int64_t workspace_bytes, void* stream) {
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
  PK_REQUIRE(nb * block < (1LL << 31) && n < (1LL << 24), "sizes out of range");
  PK_REQUIRE(cap == -1 || (cap >= 0 && (cap + block - 1) / block == nb), "cap must be the rows of the cache that the bounds are of, or -1");
  if (bs * T * H == 0) return PK_OK;
  PK_REQUIRE(nb > 0, "bounds of no block");
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255) || workspace_bytes < pk_select_blocks_workspace_bytes(bs, T, H, nb)) return fail(PK_ERR_WORKSPACE, "select_blocks: workspace missing, misaligned or too small");
  SelectParams p = {};
  p.q = (const uint16_t*)queries->data, p.q_b = queries->stride[0], p.q_t = queries->stride[1], p.q_h = queries->stride[2];
  p.bounds = (const uint16_t*)bounds->data, p.o_b = bounds->stride[0], p.o_h = bounds->stride[1], p.o_j = bounds->stride[2], p.nb = nb;
  p.cap = cap < 0 ? nb * block : cap;
  p.lengths = (const int32_t*)lengths->data, p.T = (int)T, p.H = (int)H, p.G = (int)(Hq / H), p.n = (int)n, p.block = (int)block;
  p.sink = (int)sink_blocks, p.local = (int)local_blocks, p.keys = (uint32_t*)workspace, p.ids = (int32_t*)blocks->data;
  const int64_t rows = bs * T * H;
  PK_REQUIRE(rows < (1LL << 31) && bs < 65536, "sizes out of range");
  StageTimer timer(ST_RANK, (cudaStream_t)stream);
  // tokens share what is read, four at a time; one wave where that is possible, a warp eight blocks of keys a step
  const int tt = T >= 3 ? 4 : (int)T;
  const int64_t per_head = (nb + 31) / 32, heads = H * ((T + tt - 1) / tt), slots = (int64_t)SCORE_CTAS * sm_count() / (heads * bs), room = slots < 1 ? 1 : slots;
  PK_REQUIRE(heads < 65536, "at most 65535 KV heads x token groups");
  const dim3 grid((unsigned)(per_head < room ? per_head : room), (unsigned)heads, (unsigned)bs);
  p.limits = (float*)(p.keys + rows * nb);
  auto score = [&](auto tokens) -> int {
    constexpr int TT = decltype(tokens)::value;
    static PerDevice opted;
    if (const unsigned long long bit = first_on_device(opted)) {
      if (cudaFuncSetAttribute(block_score_kernel<TT>, cudaFuncAttributeMaxDynamicSharedMemorySize, SCORE_STAGES * SCORE_STAGE) != cudaSuccess)
        return fail(PK_ERR_CUDA, "select_blocks: %s", cudaGetErrorString(cudaGetLastError()));
      mark_on_device(opted, bit);
    }
    launch_chain(block_score_kernel<TT>, grid, dim3(SCORE_THREADS), SCORE_STAGES * SCORE_STAGE, (cudaStream_t)stream, p);
    return PK_OK;
  };
  if (const int rc = tt == 1 ? score(std::integral_constant<int, 1>()) : tt == 2 ? score(std::integral_constant<int, 2>()) : score(std::integral_constant<int, 4>())) return rc;
  auto pick = [&](auto kpt) {
    launch_chain(block_pick_kernel<decltype(kpt)::value>, dim3((unsigned)rows), dim3(PICK_THREADS), 0, (cudaStream_t)stream, p, (int)grid.x * 4);
  };
  if (nb <= PICK_THREADS) pick(std::integral_constant<int, 1>());
  else if (nb <= 4 * PICK_THREADS) pick(std::integral_constant<int, 4>());
  else if (nb <= 16 * PICK_THREADS) pick(std::integral_constant<int, 16>());
  else pick(std::integral_constant<int, 0>());
  return check_launch("select_blocks", 2);
}
