// Attention of the drafted tokens of a sequence - a tree, given by a mask - over the cache and over the drafts themselves.
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(s_j - max s),  s_j = scale * log2(e) * q.k_j
// over the rows j that the query sees; a query that sees none gets zeros.
//
// The T tokens and G query heads of a KV head are the T * G rows of one product with the same keys, so that the cache is read once
// for all of them.  Tiles of 128 keys: S = Q K^T and O += P V run on tcgen05 with 128 query rows each, S, P and O in tensor memory,
// K and V by TMA into a ring of 32 KB stages.  A block is two streams of eight softmax warps (two threads per query row, half of a tile's keys each):
//   NT = 2   (more than 128 rows)  a stream per 128 query rows, both over every tile: K and V are read once for 256 rows
//   NT = 1   both streams have the same rows, one takes the even tiles and the other the odd ones
// so that while one stream's scores become probabilities the tensor cores work for the other.
// The tiles of all (sample, KV head, row group) items, laid end to end, are cut into equal ranges, one per SM; the lengths come from
// device memory, every block finds its range by itself.  Items that are cut leave partial (m, l, O) records, which tree_merge_kernel joins
// in a fixed order.
#include "tiles.cuh"

namespace pk {
namespace {

constexpr int TA_TILE = 128;                   // keys of a tile
constexpr int TA_THREADS = 576;                // two streams of eight softmax warps, a warp for the copies, a warp for the products
constexpr int TA_STAGE = 32768;                // a tile of K or V: two halves of 64 channels, 128 rows of 128 bytes
constexpr int TA_WAIT_LIMIT = 100000;          // tries; one waits up to 10 us by itself
// Up to so many query rows attend_few.cu has the call: two operands of 16 rows take its registers, one block per SM, and twice the time.  B200, us, replayed graphs, 8 KV
// heads of 4 queries, attend_few.cu | here:  701 keys, 4 rows 8.7 | 11.3, 16 rows 11.4 | 11.7, 32 rows 23.1 | 12.5;  131072 keys, 4 rows 91.2 | 92.1, 8 rows
// 92.8 | 92.3, 16 rows 95.6 | 94.3, 20 rows 175 | 94, 32 rows 202 | 97;  8 x 8192 keys, 8 rows 53.9 | 58, 16 rows 58.5 | 59, 32 rows 131 | 63.
constexpr int TA_FEW = 16;
constexpr float TA_LAZY = 8.0f;                // log2: the maximum that O is scaled to may lie this far below the true one

template <int NT> struct TaRing { static constexpr int stages = NT == 2 ? 5 : 6; };

struct TreeParams {
  AttendParams a;
  int bs;
  int tile_tokens;     // tokens of 128 query rows: 128 / G
  int row_groups;      // groups of NT * tile_tokens tokens
  int draft_tiles;
  float* records;      // [2 * blocks][rows * 130]: O rows of 128, then m, then l
};

// Tiles of an item of sample b, and where the items of a sample begin in the sequence of all tiles.
struct TreePlan {
  int64_t total;       // tiles of the launch
  int64_t before;      // tiles of the samples before `sample`
  int sample;
};
__device__ __forceinline__ int tree_len(const TreeParams& p, int b) { return (int)min((int64_t)max(p.a.lengths[b], 0), p.a.cap); }
__device__ __forceinline__ int tree_tiles(const TreeParams& p, int len) { return (len + TA_TILE - 1) / TA_TILE + p.draft_tiles; }
// By one warp: the total, and the sample that holds tile `at(total)`.
template <typename At>
__device__ __forceinline__ TreePlan tree_plan(const TreeParams& p, At at) {
  const int lane = threadIdx.x & 31;
  const int64_t items = (int64_t)p.a.H * p.row_groups;
  int64_t total = 0;
  for (int b0 = 0; b0 < p.bs; b0 += 32) {
    int n = b0 + lane < p.bs ? tree_tiles(p, tree_len(p, b0 + lane)) : 0;
    total += items * __reduce_add_sync(0xffffffffu, n);
  }
  const int64_t t = at(total);
  TreePlan r = {total, 0, 0};
  for (int b0 = 0; b0 < p.bs; b0 += 32) {
    const int64_t mine = b0 + lane < p.bs ? items * tree_tiles(p, tree_len(p, b0 + lane)) : 0;
    int64_t end = mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int64_t o = __shfl_up_sync(0xffffffffu, end, off);
      if (lane >= off) end += o;
    }
    const unsigned past = __ballot_sync(0xffffffffu, b0 + lane < p.bs && r.before + end > t);
    if (past) {
      const int i = __ffs(past) - 1;
      r.sample = b0 + i;
      r.before += __shfl_sync(0xffffffffu, end - mine, i);
      return r;
    }
    r.before += __shfl_sync(0xffffffffu, end, 31);
  }
  return r;
}

// A block's way through its range: segments of consecutive tiles of one item.
struct Cursor {
  int b, h, group, len, n, tile;   // n tiles in the item, `tile` the next
  int64_t left;                    // tiles of the range that are left
  __device__ __forceinline__ int count() const { return (int)min((int64_t)(n - tile), left); }
  __device__ __forceinline__ void next(const TreeParams& p) {
    left -= count();
    tile = 0;
    if (++group == p.row_groups) {
      group = 0;
      if (++h == p.a.H) {
        h = 0;
        if (++b < p.bs) len = tree_len(p, b), n = tree_tiles(p, len);
      }
    }
  }
};

template <int NS>
struct TreeShared {
  unsigned long long bars[2 * NS + 8];
  float most[2][2][128];   // [stream][half of the keys][row]: maxima, on their way to the other half
  TreePlan plan;
  unsigned tmem, bad[8];   // bad: drafts whose rows of V hold what is not a number
  int dead;
};

template <int NT>
__global__ void __launch_bounds__(TA_THREADS, 1)
    tree_tile_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_dk,
                     const __grid_constant__ CUtensorMap map_dv, const __grid_constant__ TreeParams p) {
  constexpr int NS = TaRing<NT>::stages;
  extern __shared__ __align__(1024) unsigned char dyn[];   // (the kernel has no other shared memory: it begins where the block's does, on such a boundary)
  TreeShared<NS>& sh = *reinterpret_cast<TreeShared<NS>*>(dyn + (NT + NS) * TA_STAGE);
  unsigned (&s_bad)[8] = sh.bad;
  volatile int& s_dead = sh.dead;
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const unsigned q_smem = smem_addr(dyn), ring = q_smem + NT * TA_STAGE;
  const unsigned full = smem_addr(sh.bars), empty = full + 8 * NS, s_full = empty + 8 * NS, p_full = s_full + 16, o_done = p_full + 16, q_full = o_done + 16, ending = q_full + 8;
  if (tid == 0) {
    for (int i = 0; i < NS; i++) mbar_init(full + 8 * i, 1), mbar_init(empty + 8 * i, 1);
    for (int i = 0; i < 2; i++) mbar_init(s_full + 8 * i, 1), mbar_init(p_full + 8 * i, 256), mbar_init(o_done + 8 * i, 1);
    mbar_init(q_full, 512), mbar_init(ending, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    s_dead = 0;
  }
  if (tid < 8) s_bad[tid] = 0;
  if (warp == 16) tmem_alloc(smem_addr(&sh.tmem), 512);
  if (warp == 17 && lane < 4) tma_prefetch_map(lane == 0 ? &map_k : lane == 1 ? &map_v : lane == 2 ? &map_dk : &map_dv);
  pdl_wait();
  pdl_trigger();
  const int blocks = (int)gridDim.x;
  if (warp == 0) {
    const TreePlan plan = tree_plan(p, [&](int64_t total) { return total * blockIdx.x / min((int64_t)blocks, total); });
    if (lane == 0) sh.plan = plan;
  }
  tc_before();
  __syncthreads();
  tc_after();
  const unsigned tmem = sh.tmem;
  const TreePlan plan = sh.plan;
  const int64_t shares = min((int64_t)blocks, plan.total);
  Cursor cur;
  {
    const int64_t first = blockIdx.x < shares ? plan.total * blockIdx.x / shares : plan.total, end = blockIdx.x < shares ? plan.total * (blockIdx.x + 1) / shares : first;
    cur.left = end - first, cur.b = plan.sample, cur.len = tree_len(p, plan.sample), cur.n = tree_tiles(p, cur.len);
    const int64_t at = first - plan.before;
    const int item = (int)(at / cur.n);
    cur.tile = (int)(at % cur.n), cur.h = item / p.row_groups, cur.group = item % p.row_groups;
  }
  // Every wait has a limit.  Where one runs out the block stops waiting altogether, its copies land, its tensor memory is freed and its
  // rows come out as NaN.
  bool dead = false;
  auto wait = [&](unsigned mb, unsigned parity) {
    for (int it = 0; !dead; it++) {
      if (mbar_try(mb, parity)) break;
      if (it >= TA_WAIT_LIMIT || ((it & 1023) == 1023 && s_dead)) dead = true, s_dead = 1;
    }
  };

  if (warp == 16) {
    // ---- copies: K and V of every tile in turn ----
    if (lane == 0) {
      unsigned q = 0;
      for (; cur.left > 0 && !dead; cur.next(p)) {
        const int n = cur.count(), cache_tiles = cur.n - p.draft_tiles;
        for (int j = 0; j < n && !dead; j++) {
          const int t = cur.tile + j;
          const bool draft = t >= cache_tiles;
          const int row = (draft ? t - cache_tiles : t) * TA_TILE;
          for (int v = 0; v < 2; v++, q++) {
            const unsigned st = q % NS;
            if (q >= NS) wait(empty + 8 * st, (q / NS - 1) & 1);
            if (dead) break;
            const CUtensorMap* map = draft ? (v ? &map_dv : &map_dk) : (v ? &map_v : &map_k);
            mbar_expect(full + 8 * st, TA_STAGE);
            tma_load4(ring + st * TA_STAGE, map, 0, row, cur.h, cur.b, full + 8 * st);
            tma_load4(ring + st * TA_STAGE + TA_STAGE / 2, map, 64, row, cur.h, cur.b, full + 8 * st);
          }
        }
      }
      if (dead || s_dead)   // what is under way has to land before the block ends
        for (unsigned i = q < NS ? 0 : q - NS; i < q; i++)
          for (int it = 0; it < TA_WAIT_LIMIT && !mbar_try(full + 8 * (i % NS), (i / NS) & 1); it++) {}
    }
  } else if (warp == 17) {
    // ---- products: the whole warp goes the same way, one lane issues.  What an instruction needs besides is a constant added to a descriptor: computed
    // anew for each, by a single thread, the descriptors took 100 clocks an instruction, which executes in 64. ----
    constexpr unsigned ID_S = umma_idesc(128, 128, false), ID_O = umma_idesc(128, 128, true), STAGE = TA_STAGE >> 4;
    const bool leader = elect_one();
    const uint64_t q_desc = umma_desc(q_smem, 16), k_desc = umma_desc(ring, 16), v_desc = umma_desc(ring, TA_STAGE / 2);
    struct Place {   // of a copy in the ring
      unsigned st, phase;
      __device__ __forceinline__ Place plus(unsigned n) const { return st + n < NS ? Place{st + n, phase} : Place{st + n - NS, phase ^ 1}; }
    };
    auto scores = [&](int s, Place k) {   // S_s = Q K^T
      const uint64_t a = q_desc + (NT == 2 ? s * STAGE : 0u), b = k_desc + k.st * STAGE;
      if (leader && !dead) {
        tc_mma_ss<false>(tmem + 128 * s, a, b, ID_S);
#pragma unroll
        for (int i = 1; i < 8; i++) {
          const unsigned off = ((i >> 2) * (TA_STAGE / 2) + (i & 3) * 32) >> 4;
          tc_mma_ss<true>(tmem + 128 * s, a + off, b + off, ID_S);
        }
        tc_commit(s_full + 8 * s);
      }
    };
    auto values = [&](int s, Place v, bool add) {   // O_s (+)= P_s V
      const uint64_t b = v_desc + v.st * STAGE;
      if (leader && !dead) {
#pragma unroll
        for (int i = 0; i < 8; i++) tc_mma_ts(tmem + 256 + 128 * s, tmem + 128 * s + 64 * (i >> 2) + 8 * (i & 3), b + i * (2048 >> 4), ID_O, i > 0 ? 1u : (unsigned)add);
      }
    };
    auto commit = [&](unsigned mb) {
      if (leader && !dead) tc_commit(mb);
    };
    auto free_stage = [&](Place at) { commit(empty + 8 * at.st); };
    auto arrived = [&](Place at) {
      wait(full + 8 * at.st, at.phase);
      __syncwarp();
      tc_after();
    };
    unsigned n_p[2] = {0, 0}, seg = 0;
    auto probabilities = [&](int s) {
      wait(p_full + 8 * s, n_p[s] & 1);
      n_p[s] ^= 1;
      __syncwarp();
      tc_after();
    };
    Place at = {0, 0};   // of the tile's K
    for (; cur.left > 0; cur.next(p), seg ^= 1) {
      const int n = cur.count();
      wait(q_full, seg);
      __syncwarp();
      tc_after();
      arrived(at);
      scores(0, at);
      if (NT == 2) scores(1, at);
      free_stage(at);
      if (NT == 1 && n > 1) {
        arrived(at.plus(2));
        scores(1, at.plus(2));
        free_stage(at.plus(2));
      }
      for (int j = 0; j < n; j++, at = at.plus(2)) {
        const Place v = at.plus(1), k_next = at.plus(NT == 2 ? 2 : 4);
        const bool more = j + (NT == 2 ? 1 : 2) < n;
        arrived(v);
#pragma unroll
        for (int i = 0; i < NT; i++) {
          const int s = NT == 2 ? i : j & 1;
          probabilities(s);
          values(s, v, NT == 2 ? j > 0 : j > 1);
          if (i == NT - 1) free_stage(v);
          if (more) {
            if (i == 0) arrived(k_next);
            scores(s, k_next);
            if (i == NT - 1) free_stage(k_next);
          } else {
            commit(o_done + 8 * s);
          }
        }
      }
    }
    if (s_dead && leader) {   // products under way end before the tensor memory goes
      tc_commit(ending);
      for (int it = 0; it < TA_WAIT_LIMIT && !mbar_try(ending, 0); it++) {}
    }
  } else {
    // ---- softmax: stream `s`, two threads per query row: `part` is the half of a tile's keys, and of the channels of O ----
    const int s = warp >> 3, part = warp >> 2 & 1, r = 32 * (warp & 3) + lane;
    const unsigned lanes = tmem + ((unsigned)(warp & 3) << 21), s_cols = lanes + 128 * s + 64 * part, o_cols = lanes + 256;   // this half's scores, and its weights in their place
    const int pair = 3 + 4 * s + (warp & 3);   // barrier of the two warps that share rows
    const int Hq = p.a.H * p.a.G, tl = r / p.a.G, g = r % p.a.G;
    const float scale = p.a.scale_log2;
    unsigned q0 = 0, n_s = 0, n_o[2] = {0, 0};
    for (; cur.left > 0; cur.next(p)) {
      const int n = cur.count(), cache_tiles = cur.n - p.draft_tiles;
      const int token0 = (NT == 2 ? 2 * cur.group + s : cur.group) * p.tile_tokens, t = token0 + tl;
      const bool row_ok = tl < p.tile_tokens && t < p.a.T;
      const bool warp_ok = __any_sync(0xffffffffu, row_ok);
      {  // this thread's share of its row of Q, swizzled as the copies of K are
        constexpr int CHUNKS = NT == 2 ? 8 : 4;
        const int half = NT == 2 ? part : s, c0 = NT == 2 ? 0 : 4 * part;
        const uint16_t* src = p.a.q + cur.b * p.a.q_b + (int64_t)t * p.a.q_t + (int64_t)(cur.h * p.a.G + g) * p.a.q_h + half * 64 + 8 * c0;
        const unsigned dst = q_smem + (NT == 2 ? s * TA_STAGE : 0) + half * (TA_STAGE / 2) + r * 128;
        uint4 x[CHUNKS];
#pragma unroll
        for (int c = 0; c < CHUNKS; c++) x[c] = row_ok ? *reinterpret_cast<const uint4*>(src + 8 * c) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int c = 0; c < CHUNKS; c++)
          asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(dst + (((c0 + c) ^ (r & 7)) << 4)), "r"(x[c].x), "r"(x[c].y), "r"(x[c].z), "r"(x[c].w) : "memory");
        fence_async();
        mbar_arrive1(q_full);
      }
      // which drafts of draft tile dt this row sees: a token's bytes by 32 lanes at a time
      auto drafts_seen = [&](int dt, uint32_t (&w)[2]) {
        const int t_first = token0 + (32 * (warp & 3)) / p.a.G, t_last = min(token0 + (32 * (warp & 3) + 31) / p.a.G, p.a.T - 1);
        const uint8_t* mask = p.a.mask + cur.b * p.a.m_b;
#pragma unroll
        for (int i = 0; i < 2; i++) {
          const int d = dt * TA_TILE + 64 * part + 32 * i + lane;
          w[i] = 0;
          if (d - lane < p.a.T)
#pragma unroll 4
            for (int tt = t_first; tt <= t_last; tt++) {
              const unsigned bits = __ballot_sync(0xffffffffu, d < p.a.T && mask[tt * p.a.m_t + d * p.a.m_j] != 0);
              if (tt == t) w[i] = bits;
            }
        }
      };
      uint32_t drafts[2] = {};
      if (cur.tile + n > cache_tiles && cur.tile <= cache_tiles) drafts_seen(0, drafts);
      float m = -INFINITY, l = 0.0f;   // m: raw scores
      for (int j = NT == 2 ? 0 : s; j < n; j += NT == 2 ? 1 : 2) {
        const int tile = cur.tile + j, dt = tile - cache_tiles;
        const int live = dt >= 0 ? TA_TILE : cur.len - tile * TA_TILE;
        uint32_t w[2] = {~0u, ~0u};
        if (dt == 0) {
          w[0] = drafts[0], w[1] = drafts[1];
        } else if (dt > 0) {
          drafts_seen(dt, w);
        } else if (live < TA_TILE) {
#pragma unroll
          for (int i = 0; i < 2; i++) {
            const int n_live = live - 64 * part - 32 * i;
            w[i] = n_live >= 32 ? ~0u : n_live <= 0 ? 0u : (1u << n_live) - 1;
          }
        }
        const bool masked = dt >= 0 || live < TA_TILE;
        wait(s_full + 8 * s, n_s & 1);
        n_s++;
        __syncwarp();
        tc_after();
        if (warp_ok) {
          // The scores are read twice, for the maximum and for the weights.
          auto masked_scores = [&](int c, uint32_t (&x)[32]) {
            wait_ld(x);
            if (masked) {
#pragma unroll
              for (int i = 0; i < 32; i++) x[i] = w[c] >> i & 1 ? x[i] : 0xff800000u;
            }
          };
          float mx[4] = {m, m, m, m};
          {
            uint32_t x[2][32];
            tmem_ld32(x[0], s_cols);
            tmem_ld32(x[1], s_cols + 32);
#pragma unroll
            for (int c = 0; c < 2; c++) {
              masked_scores(c, x[c]);
#pragma unroll
              for (int i = 0; i < 32; i += 8)
#pragma unroll
                for (int e = 0; e < 4; e++) mx[e] = max3(mx[e], __uint_as_float(x[c][i + 2 * e]), __uint_as_float(x[c][i + 2 * e + 1]));
            }
          }
          const float mine = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
          sh.most[s][part][r] = mine;
          named_barrier(pair, 64);
          const float m_new = fmaxf(mine, sh.most[s][part ^ 1][r]);
          if (j < 2 - (NT == 2)) {   // the stream's first tile: nothing to scale
            m = m_new;
          } else {
            const bool grow = (m_new - m) * scale > TA_LAZY;
            if (__any_sync(0xffffffffu, grow)) {
              const float f = grow ? ex2((m - m_new) * scale) : 1.0f;
              if (grow) m = m_new;
              l *= f;
              // the products of the tile before have ended: their commit came before that of these scores
#pragma unroll
              for (int c = 2 * part; c < 2 * part + 2; c++) {
                uint32_t o[32];
                tmem_ld32(o, o_cols + 128 * s + 32 * c);
                wait_ld(o);
#pragma unroll
                for (int i = 0; i < 32; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                tmem_st32(o_cols + 128 * s + 32 * c, o);
              }
            }
          }
          const float least = m == -INFINITY ? 0.0f : -m;   // (x - m) scale, not x scale - m scale: the difference of close scores is exact
          // Weights meet V as bf16, 8 bits: a tcgen05 product of bf16 values takes no others; the sums have all of their bits.  That is 0.0009 to 0.0014 of the
          // outputs' norm beside the 0.0016 that their own rounding to bf16 is (both against 64 bits: 0.0016 to 0.0018).  What the rounding leaves as a
          // second product, as attend_few.cu has it for eight rows, made it 0.0002, and 61 tokens over 128K keys 182 -> 219 us, 26 over 64K 99 -> 117.
          float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};   // two pairs
#pragma unroll
          for (int c = 0; c < 2; c++) {
            uint32_t x[32], pr[16];
            tmem_ld32(x, s_cols + 32 * c);
            masked_scores(c, x);
            // sixteen at a time, step by step, so that no step waits for the one before
#pragma unroll
            for (int i0 = 0; i0 < 32; i0 += 16) {
              float y[16];
#pragma unroll
              for (int i = 0; i < 16; i++) y[i] = __uint_as_float(x[i0 + i]);
#pragma unroll
              for (int i = 0; i < 16; i += 2) add_mul2(y[i], y[i + 1], least, scale);
#pragma unroll
              for (int i = 0; i < 16; i++) y[i] = ex2(y[i]);
#pragma unroll
              for (int i = 0; i < 16; i += 2) {
                add2(sum[i & 2], sum[(i & 2) + 1], y[i], y[i + 1]);
                pr[(i0 + i) / 2] = pack2(y[i], y[i + 1]);
              }
            }
            tmem_st16(s_cols + 16 * c, pr);
          }
          l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
          tmem_wait_st();
        }
        if (masked) {
          // rows of V that no query sees must be zero, what is not a number in a draft's row must not reach the queries that do not see
          // it: a weight of zero would not keep it out of the product.  Half a row a thread.
          const unsigned vq = q0 + 2 * j + 1, row = ring + (vq % NS) * TA_STAGE + part * (TA_STAGE / 2) + r * 128;
          wait(full + 8 * (vq % NS), (vq / NS) & 1);
          if (dt < 0) {
            if (r >= live)
#pragma unroll
              for (int c = 0; c < 8; c++) asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(row + c * 16), "r"(0) : "memory");
          } else {
            bool bad = false;
#pragma unroll 4
            for (int c = 0; c < 8; c++) {
              const unsigned at = row + c * 16;
              uint32_t v[4];
              asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(at) : "memory");
              bool here = false;
#pragma unroll
              for (int i = 0; i < 4; i++) here |= not_finite(v[i]) | not_finite(v[i] >> 16);
              if (here) {
                if (!bad) atomicOr(&s_bad[4 * dt + (r >> 5)], 1u << (r & 31)), __threadfence_block();
                bad = true;
#pragma unroll
                for (int i = 0; i < 4; i++) v[i] = (not_finite(v[i]) ? 0 : v[i] & 0xffffu) | (not_finite(v[i] >> 16) ? 0 : v[i] & 0xffff0000u);
                asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
              }
            }
          }
          fence_async();
        }
        tc_before();
        mbar_arrive1(p_full + 8 * s);
      }
      // ---- the segment's result ----
      const bool whole = cur.tile == 0 && n == cur.n;
      const int64_t out_row = ((int64_t)cur.b * p.a.T + t) * Hq + cur.h * p.a.G + g;
      float* rec = nullptr;
      constexpr int ROWS = NT * 128;
      const int rec_row = NT == 2 ? s * 128 + r : r;
      if (!whole) rec = p.records + (2 * (int64_t)blockIdx.x + (cur.tile == 0)) * (ROWS * 130);
      const bool two = NT == 1 && n > 1;   // both streams have tiles of this segment
      float f[2] = {1.0f, 1.0f}, M = m == -INFINITY ? -INFINITY : m * scale, L = l;
      wait(o_done + 8 * (NT == 2 ? s : 0), n_o[0]++ & 1);
      if (two) wait(o_done + 8, n_o[1]++ & 1);
      __syncwarp();
      tc_after();
      {  // maxima and sums of both halves of the keys (NT = 1: and of both streams), through the room of Q
        const unsigned at = q_smem + (NT == 2 ? s * TA_STAGE : 0) + r * 8;
        asm volatile("st.shared.v2.b32 [%0], {%1,%2};" ::"r"(at + ((NT == 2 ? 0 : 2 * s) + part) * 1024), "f"(M), "f"(L) : "memory");
        named_barrier(NT == 2 ? pair : 1, NT == 2 ? 64 : 512);
        float m2[2 / NT], l2[2 / NT];
#pragma unroll
        for (int i = 0; i < 2 / NT; i++) {
          float again, more;
          asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=f"(m2[i]), "=f"(l2[i]) : "r"(at + 2 * i * 1024) : "memory");
          asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=f"(again), "=f"(more) : "r"(at + (2 * i + 1) * 1024) : "memory");
          l2[i] += more;
        }
        M = NT == 2 ? m2[0] : fmaxf(m2[0], m2[2 / NT - 1]), L = 0.0f;
#pragma unroll
        for (int i = 0; i < 2 / NT; i++) {
          f[i] = m2[i] == -INFINITY ? 0.0f : NT == 2 ? 1.0f : ex2(m2[i] - M);
          L += l2[i] * f[i];   // (of a stream without tiles: m = -inf, l = 0)
        }
      }
      if (dead) L = NAN;
      if (warp_ok) {
        const float inv = L == 0.0f ? 0.0f : 1.0f / L;
#pragma unroll
        for (int c = 0; c < 4; c++) {
          if (NT == 2 ? (c >> 1) != part : c != 2 * s + part) continue;   // this thread's channels
          uint32_t o[32];
          tmem_ld32(o, o_cols + (NT == 2 ? 128 * s : 0) + 32 * c);
          wait_ld(o);
          if (two) {
            uint32_t o1[32];
            tmem_ld32(o1, o_cols + 128 + 32 * c);
            wait_ld(o1);
#pragma unroll
            for (int i = 0; i < 32; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * f[0] + __uint_as_float(o1[i]) * f[1]);
          }
          // what was taken out of the drafts' rows, back to the queries that see it
          if (s_bad[0] | s_bad[1] | s_bad[2] | s_bad[3] | s_bad[4] | s_bad[5] | s_bad[6] | s_bad[7]) {
            const int d_first = max(cur.tile - cache_tiles, 0) * TA_TILE, d_end = min(p.a.T, (cur.tile + n - cache_tiles) * TA_TILE);
            const uint8_t* mask = p.a.mask + cur.b * p.a.m_b + (int64_t)(row_ok ? t : 0) * p.a.m_t;
            for (int d = d_first; d < d_end; d++)
              if (row_ok && mask[d * p.a.m_j]) {
                const uint16_t* v = p.a.dv + cur.b * p.a.dv_b + (int64_t)d * p.a.dv_t + cur.h * p.a.dv_h + 32 * c;
#pragma unroll
                for (int i = 0; i < 32; i++)
                  if (not_finite(v[i])) o[i] = __float_as_uint(__uint_as_float(o[i]) + bf2f(v[i]));
              }
          }
          if (row_ok) {
            if (whole) {
              uint4* dst = reinterpret_cast<uint4*>(p.a.out + out_row * 128 + 32 * c);
#pragma unroll
              for (int i = 0; i < 4; i++) {
                uint32_t y[4];
#pragma unroll
                for (int e = 0; e < 4; e++) y[e] = pack2(__uint_as_float(o[8 * i + 2 * e]) * inv, __uint_as_float(o[8 * i + 2 * e + 1]) * inv);
                dst[i] = make_uint4(y[0], y[1], y[2], y[3]);
              }
            } else {
              float* dst = rec + (int64_t)rec_row * 128 + 32 * c;
#pragma unroll
              for (int i = 0; i < 32; i += 8)   // whole sectors
                asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(dst + i), "r"(o[i]), "r"(o[i + 1]), "r"(o[i + 2]), "r"(o[i + 3]), "r"(o[i + 4]),
                             "r"(o[i + 5]), "r"(o[i + 6]), "r"(o[i + 7])
                             : "memory");
            }
          }
        }
        if (row_ok && part == 0 && (NT == 2 || s == 0)) {
          if (whole) {
            if (p.a.lse) p.a.lse[out_row] = L == 0.0f ? -INFINITY : M + log2f(L);
          } else {
            rec[ROWS * 128 + rec_row] = M, rec[ROWS * 129 + rec_row] = L;
          }
        }
      }
      tc_before();
      named_barrier(2, 512);   // both streams have read: the room of Q, O and the marks may be written
      if (tid < 8) s_bad[tid] = 0;
      q0 += 2 * n;
    }
  }
  __syncwarp();
  tc_before();
  __syncthreads();
  tc_after();
  if (warp == 16) tmem_free(tmem, 512);
}

// A block per query row: the records of the blocks that share its item, in the order of the tiles.
template <int NT>
__global__ void __launch_bounds__(128) tree_merge_kernel(const __grid_constant__ TreeParams p, int blocks) {
  pdl_wait();
  pdl_trigger();
  __shared__ MergeShared shared;
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x & 31, Hq = p.a.H * p.a.G, hq = (int)(row % Hq), h = hq / p.a.G, g = hq % p.a.G;
  const int b = (int)(row / Hq / p.a.T), t = (int)(row / Hq % p.a.T), mt = t / p.tile_tokens, group = mt / NT;
  const int r = (mt % NT) * 128 + (t - mt * p.tile_tokens) * p.a.G + g;
  const int64_t items = (int64_t)p.a.H * p.row_groups;
  int64_t total = 0, before = 0;
  for (int b0 = 0; b0 < p.bs; b0 += 32) {
    const int n = b0 + lane < p.bs ? tree_tiles(p, tree_len(p, b0 + lane)) : 0;
    total += items * __reduce_add_sync(0xffffffffu, n), before += items * __reduce_add_sync(0xffffffffu, b0 + lane < b ? n : 0);
  }
  const int n = tree_tiles(p, tree_len(p, b));
  const int64_t first = before + ((int64_t)h * p.row_groups + group) * n, last = first + n - 1;
  const unsigned shares = (unsigned)min((int64_t)blocks, total);
  const int c0 = share_owner(first, total, shares), c1 = share_owner(last, total, shares);
  if (c0 == c1) return;   // written by its block
  constexpr int ROWS = NT * 128;
  merge_row(shared, c1 - c0 + 1, ROWS, r, [&](int i) { return p.records + (2 * (int64_t)(c0 + i) + (i == 0)) * (ROWS * 130); }, p.a.out + row * 128, p.a.lse ? p.a.lse + row : nullptr);
}

template <int NT>
int launch_tree(const AttendParams& a, int64_t bs, void* workspace, cudaStream_t st) {
  CUtensorMap mk, mv, mdk, mdv;
  if (!rows_map(&mk, a.k, a.cap, a.k_l, a.H, a.k_h, bs, a.k_b, TA_TILE) || !rows_map(&mv, a.v, a.cap, a.v_l, a.H, a.v_h, bs, a.v_b, TA_TILE) ||
      !rows_map(&mdk, a.dk, a.T, a.dk_t, a.H, a.dk_h, bs, a.dk_b, TA_TILE) || !rows_map(&mdv, a.dv, a.T, a.dv_t, a.H, a.dv_h, bs, a.dv_b, TA_TILE))
    return launch_attend_rows(a, bs, "tree_attention", st);
  TreeParams p = {};
  p.a = a, p.bs = (int)bs, p.tile_tokens = 128 / a.G, p.row_groups = (a.T + NT * p.tile_tokens - 1) / (NT * p.tile_tokens);
  p.draft_tiles = (a.T + TA_TILE - 1) / TA_TILE, p.records = (float*)workspace;
  const int64_t most = bs * a.H * p.row_groups * ((a.cap + TA_TILE - 1) / TA_TILE + p.draft_tiles);
  const int blocks = (int)(most < sm_count() ? most : sm_count());
  static PerDevice opted;
  constexpr int SMEM = (NT + TaRing<NT>::stages) * TA_STAGE + (int)sizeof(TreeShared<TaRing<NT>::stages>);
  static_assert(SMEM <= 227 * 1024, "shared memory of a block");
  if (const unsigned long long bit = first_on_device(opted)) {
    if (cudaFuncSetAttribute(tree_tile_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM) != cudaSuccess)
      return fail(PK_ERR_CUDA, "tree_attention: %s", cudaGetErrorString(cudaGetLastError()));
    mark_on_device(opted, bit);
  }
  StageTimer timer(ST_ATTENTION, st);
  launch_chain(tree_tile_kernel<NT>, dim3((unsigned)blocks), dim3(TA_THREADS), SMEM, st, mk, mv, mdk, mdv, p);
  const int64_t rows = bs * a.T * a.H * a.G;
  launch_chain(tree_merge_kernel<NT>, dim3((unsigned)rows), dim3(128), 0, st, p, blocks);
  return check_launch("tree_attention", 2);
}

}  // namespace
}  // namespace pk

using namespace pk;

extern "C" int64_t pk_tree_attention_workspace_bytes(int64_t, int64_t T, int64_t Hq, int64_t H, int64_t) {
  const int64_t rows = H > 0 && T * (Hq / H) > 128 ? 256 : 128;
  if (H > 0 && T * (Hq / H) <= TA_FEW) return attend_few_workspace();
  return 2 * (int64_t)sm_count() * rows * 130 * 4;
}

extern "C" int pk_tree_attention(const pk_tensor* queries, const pk_tensor* keys, const pk_tensor* values, const pk_tensor* draft_keys,
                                 const pk_tensor* draft_values, const pk_tensor* tree_mask, const pk_tensor* lengths, float scale,
                                 const pk_tensor* out, const pk_tensor* lse, void* workspace, int64_t workspace_bytes, void* stream) {
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
  if (bs == 0 || p.T == 0) return PK_OK;
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255) || workspace_bytes < pk_tree_attention_workspace_bytes(bs, p.T, queries->shape[2], p.H, p.cap))
    return fail(PK_ERR_WORKSPACE, "tree_attention: workspace missing, misaligned or too small");
  if (p.T * p.G <= TA_FEW) return launch_attend_few(p, bs, workspace, "tree_attention", (cudaStream_t)stream);
  return p.T * p.G > 128 ? launch_tree<2>(p, bs, workspace, (cudaStream_t)stream) : launch_tree<1>(p, bs, workspace, (cudaStream_t)stream);
}
