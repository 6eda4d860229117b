// Attention of a few query rows per KV head - a token over the blocks that it selected, up to 16 rows of drafted tokens over the cache - with
// the keys spread over the warps:  o = sum_j p_j v_j / sum_j p_j,  p_j = 2^((s_j - max s) scale log2 e),  s_j = q.k_j.
//
// 1 to 32 rows cannot fill the 128 rows of a tcgen05 product, and a softmax thread per row would leave most threads idle: here a warp takes
// 16 of a tile's 64 keys for all rows (mma.sync m16n8k16), its fragments of S are the operand of P V, and the four warps' (m, l, O) meet once per
// segment.  K and V come by TMA, a box per block of keys and half of the channels, three tiles of 32 KB under way in each of two blocks per SM:
// the copies, not the products, are what bounds it.  As in tree_attention.cu the tiles of all items, laid end to end, are cut into equal
// ranges, and few_merge_kernel joins the records of items that are cut.
#include "tiles.cuh"

namespace pk {
namespace {

constexpr int FEW_TILE = 64, FEW_BUFS = 3, FEW_THREADS = 160;   // four warps that share the keys, one that makes the copies
constexpr int FEW_STAGE = 32768;                    // K 64 x 128, V 64 x 128: halves of 64 channels, rows of 128 bytes
constexpr int FEW_OS = 136;                         // floats between two rows of a warp's partial: its stores fall into all banks
constexpr int FEW_SMEM = 1024 + FEW_BUFS * FEW_STAGE;
static_assert(4 * 8 * FEW_OS * 4 <= FEW_STAGE, "the warps' partials of eight rows take the place of a tile");
constexpr int FEW_WAIT_LIMIT = 100000;              // (a try waits up to 10 us by itself)

constexpr int FEW_CTAS = 2;                         // blocks per SM: by the registers

struct FewParams {
  AttendParams a;
  int bs;
  int row_groups;     // groups of query rows of an item (blocks: of one token; tree: one)
  int tiles;          // blocks: tiles of an item
  int box;            // keys of a copy
  float* records;     // [2 * blocks][rows * 130]
};

struct TilePlan {
  int64_t total;    // tiles of the launch
  int64_t before;   // tiles of the samples before `sample`
  int sample;
};
// By a whole warp: the total, and the sample that holds tile share_begin(total, block, min(blocks, total)); tiles_of(b): tiles of sample b, 0 behind the last.
template <class TilesOf>
__device__ __forceinline__ TilePlan tile_plan(int bs, unsigned block, unsigned blocks, TilesOf tiles_of) {
  const int lane = threadIdx.x & 31;
  const int64_t first = tiles_of(lane);
  TilePlan r = {0, 0, 0};
  auto sum = [](int64_t v) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    return v;
  };
  r.total = sum(first);
  for (int b0 = 32; b0 < bs; b0 += 32) r.total += sum(tiles_of(b0 + lane));
  const int64_t t = share_begin(r.total, block, (unsigned)min((int64_t)blocks, r.total));
  for (int b0 = 0; b0 < bs; b0 += 32) {
    const int64_t mine = b0 == 0 ? first : tiles_of(b0 + lane);
    int64_t end = mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int64_t o = __shfl_up_sync(0xffffffffu, end, off);
      if (lane >= off) end += o;
    }
    const unsigned past = __ballot_sync(0xffffffffu, b0 + lane < bs && r.before + end > t);
    if (past) {
      const int i = __ffs(past) - 1;
      r.sample = b0 + i, r.before += __shfl_sync(0xffffffffu, end - mine, i);
      return r;
    }
    r.before += __shfl_sync(0xffffffffu, end, 31);
  }
  return r;
}

__device__ __forceinline__ int few_len(const FewParams& p, int b) { return (int)min((int64_t)max(p.a.lengths[b], 0), p.a.cap); }

__device__ __forceinline__ int few_tiles(const FewParams& p, int b) {   // of a tree's item
  return (few_len(p, b) + FEW_TILE - 1) / FEW_TILE + 1;
}

// A way through consecutive tiles.
template <bool TREE>
struct FewCursor {
  int b, t, h, group, len, n, tile;   // len: rows of the cache (tree), rows up to the token's position (blocks)
  __device__ __forceinline__ void sample(const FewParams& p) {
    const int rows = few_len(p, b);
    if (TREE) len = rows, n = few_tiles(p, b);
    else len = max(rows - p.a.T + t + 1, 0), n = p.tiles;
  }
  __device__ __forceinline__ void start(const FewParams& p, const TilePlan& w, int64_t first) {
    if (TREE) {
      b = w.sample, t = 0, group = 0;
      sample(p);
      const int at = (int)(first - w.before);
      h = min(at / n, p.a.H - 1), tile = at % n;
    } else {
      const int64_t item = first / p.tiles;
      tile = (int)(first - item * p.tiles);
      group = (int)(item % p.row_groups);
      const int64_t bth = item / p.row_groups;
      h = (int)(bth % p.a.H), t = (int)(bth / p.a.H % p.a.T), b = (int)(bth / p.a.H / p.a.T);
      if (b < p.bs) sample(p);
    }
  }
  __device__ __forceinline__ void step(const FewParams& p) {   // the next tile
    if (++tile < n) return;
    tile = 0;
    if (++group < p.row_groups) return;
    group = 0;
    if (++h < p.a.H) return;
    h = 0;
    if (!TREE && ++t < p.a.T) return sample(p);
    t = 0;
    if (++b < p.bs) sample(p);
  }
};

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], unsigned addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4t(uint32_t (&r)[4], unsigned addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

__device__ __forceinline__ bool finite(float x) { return fabsf(x) < INFINITY; }

// ROWS 8: the eight rows are the upper half of the A operands; in P V the lower half carries what the rounding of P to bf16 left, and the two halves
// of O are added, where that one is finite: 17 bits of each weight for no further product.  ROWS 16: a full operand, weights of 8 bits; the sums have them
// all.  More heads of a listed block are groups of 16: two operands at once took the registers of one of the two blocks per SM.  B200, us, groups of 16 | two
// operands: 16 sequences x 8 x 20 heads over 32 blocks of 64 keys 47 | 55, 4 sequences x 128 heads over 64 blocks 21 | 29, one sequence x 8 x 32 12 | 15.
template <bool TREE, int ROWS>
__global__ void __launch_bounds__(FEW_THREADS, FEW_CTAS)
    attend_few_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_dk,
                      const __grid_constant__ CUtensorMap map_dv, const __grid_constant__ FewParams p) {
  constexpr bool PAIR = ROWS == 8;
  constexpr int RPT = PAIR ? 1 : 2;               // rows of an operand that a lane's fragments belong to
  extern __shared__ unsigned char dyn[];
  __shared__ __align__(8) unsigned long long bars[2 * FEW_BUFS];
  __shared__ float s_m[4][ROWS], s_l[4][ROWS];
  __shared__ unsigned char s_live[FEW_BUFS][4];   // keys of each warp's sixteen that are seen (tree: by all tokens)
  __shared__ uint32_t s_mask[32], s_bad;
  __shared__ volatile int s_dead;
  __shared__ TilePlan s_place;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  const unsigned base = (smem_addr(dyn) + 1023) & ~1023u, full = smem_addr(bars), empty = full + 8 * FEW_BUFS;
  if (tid == 0) {
    for (int i = 0; i < FEW_BUFS; i++) mbar_init(full + 8 * i, 1), mbar_init(empty + 8 * i, 4);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    s_dead = 0, s_bad = 0;
  }
  if (tid < (TREE ? 4 : 2)) tma_prefetch_map(tid == 0 ? &map_k : tid == 1 ? &map_v : tid == 2 ? &map_dk : &map_dv);
  pdl_wait();
  pdl_trigger();
  const int blocks = (int)gridDim.x;
  if (TREE && warp == 0) {
    const TilePlan w = tile_plan(p.bs, blockIdx.x, (unsigned)blocks, [&](int b) -> int64_t { return b < p.bs ? (int64_t)p.a.H * few_tiles(p, b) : 0; });
    if (lane == 0) s_place = w;
  }
  __syncthreads();   // the barriers are there, and the place
  const TilePlan place = TREE ? s_place : TilePlan{(int64_t)p.bs * p.a.T * p.a.H * p.row_groups * p.tiles, 0, 0};
  const unsigned shares = (unsigned)min((int64_t)blocks, place.total);
  if (blockIdx.x >= shares) return;
  const int64_t first = share_begin(place.total, blockIdx.x, shares);
  const int count = (int)(share_begin(place.total, blockIdx.x + 1, shares) - first);
  FewCursor<TREE> cur;
  cur.start(p, place, first);

  bool dead = false;   // a wait has run out: no more waiting, the rows come out as NaN
  auto wait = [&](unsigned mb, unsigned parity) {
    for (int it = 0; !dead; it++) {
      if (mbar_try(mb, parity)) break;
      if (it >= FEW_WAIT_LIMIT || s_dead) dead = true, s_dead = 1;
    }
    __syncwarp();
  };

  if (warp == 4) {
    // ---- copies: a lane per box of keys ----
    const int per = TREE ? 1 : FEW_TILE / p.box;   // boxes of a tile
    int issued = 0;
    // the block of this lane's box of the tile that `cur` is at
    auto listed = [&]() -> int {
      const int i = TREE ? 0 : (cur.tile * FEW_TILE + lane * p.box) / p.a.block;
      return !TREE && lane < per && i < p.a.n ? p.a.blocks[(((int64_t)cur.b * p.a.T + cur.t) * p.a.H + cur.h) * p.a.n + i] : -1;
    };
    int id = listed();
    for (; issued < count; issued++) {
      const int buf = issued % FEW_BUFS;
      const unsigned dst = base + buf * FEW_STAGE, mb = full + 8 * buf;
      if (issued >= FEW_BUFS) wait(empty + 8 * buf, (unsigned)(issued / FEW_BUFS - 1) & 1);
      if (__any_sync(0xffffffffu, dead)) break;
      int row = 0, live = 0;   // this lane's box: first row, rows that are seen
      const bool draft = TREE && cur.tile == cur.n - 1;
      if (TREE) {
        row = draft ? 0 : cur.tile * FEW_TILE;
        live = lane > 0 ? 0 : draft ? p.a.T : min(FEW_TILE, cur.len - row);
      } else if (id >= 0) {
        const int64_t r = (int64_t)id * p.a.block + (cur.tile * FEW_TILE + lane * p.box) % p.a.block;
        live = (int)max((int64_t)0, min((int64_t)p.box, cur.len - r));
        row = (int)(live > 0 ? r : 0);
      }
      // a warp's sixteen keys lie in one box
      const int box_of = TREE ? 0 : lane * 16 / p.box, off = TREE ? lane * 16 : lane * 16 % p.box;
      const int l = __shfl_sync(0xffffffffu, live, box_of & 31);
      if (lane < 4) s_live[buf][lane] = (unsigned char)max(0, min(16, l - off));
      const unsigned boxes = __popc(__ballot_sync(0xffffffffu, live > 0));
      const unsigned keys = draft ? 32 : TREE ? FEW_TILE : p.box;
      __syncwarp();
      if (lane == 0) mbar_expect(mb, boxes * keys * 512);
      __syncwarp();
      if (live > 0) {
        const CUtensorMap *mk = draft ? &map_dk : &map_k, *mv = draft ? &map_dv : &map_v;
#pragma unroll
        for (int half = 0; half < 2; half++) {
          const unsigned to = dst + half * (FEW_STAGE / 4) + lane * p.box * 128;
          tma_load4(to, mk, 64 * half, row, cur.h, cur.b, mb);
          tma_load4(to + FEW_STAGE / 2, mv, 64 * half, row, cur.h, cur.b, mb);
        }
      }
      if (issued + 1 < count) {
        cur.step(p);
        id = listed();
      }
    }
    if (s_dead)   // what is under way has to land before the block ends
      for (int i = issued < FEW_BUFS ? 0 : issued - FEW_BUFS; i < issued; i++)
        for (int it = 0; it < FEW_WAIT_LIMIT && !mbar_try(full + 8 * (i % FEW_BUFS), (unsigned)(i / FEW_BUFS & 1)); it++) {}
    return;
  }

  const int Hq = p.a.H * p.a.G;
  const float scale = p.a.scale_log2;
  // row r of the item -> token and query head
  auto row_token = [&](int r) { return TREE ? r / p.a.G : cur.t; };
  auto row_head = [&](int r) { return cur.h * p.a.G + (TREE ? r % p.a.G : cur.group * ROWS + r); };
  const int tree_rows = p.a.T * p.a.G;
  for (int k = 0; k < count;) {
    // ---- a segment: consecutive tiles of one item ----
    const int n_rows = TREE ? tree_rows : min(ROWS, p.a.G - cur.group * ROWS);
    const int seg_first = cur.tile, seg = min(cur.n - cur.tile, count - k);
    const bool whole = seg == cur.n, has_drafts = TREE && seg_first + seg == cur.n;
    uint32_t qa[8][2 * RPT];
#pragma unroll
    for (int e = 0; e < RPT; e++) {
      const int r = 8 * e + g;
      const bool ok = r < n_rows;
      const uint32_t* q = reinterpret_cast<const uint32_t*>(p.a.q + cur.b * p.a.q_b + (ok ? (int64_t)row_token(r) * p.a.q_t + (int64_t)row_head(r) * p.a.q_h : 0));
#pragma unroll
      for (int ks = 0; ks < 8; ks++) {
        qa[ks][e] = ok ? q[8 * ks + t4] : 0u;             // columns 2 t4 of the step
        qa[ks][RPT + e] = ok ? q[8 * ks + 4 + t4] : 0u;   // and eight further
      }
    }
    if (has_drafts) {   // a bit per draft for every token
      for (int t = warp; t < p.a.T; t += 4) {
        const unsigned bits = __ballot_sync(0xffffffffu, lane < p.a.T && p.a.mask[cur.b * p.a.m_b + t * p.a.m_t + lane * p.a.m_j] != 0);
        if (lane == 0) s_mask[t] = bits;
      }
      named_barrier(1, 128);
    }
    float o[16][4] = {}, m[RPT], l[RPT];
#pragma unroll
    for (int e = 0; e < RPT; e++) m[e] = -INFINITY, l[e] = 0.0f;
    for (int j = 0; j < seg; j++, k++) {
      const int buf = k % FEW_BUFS;
      wait(full + 8 * buf, (unsigned)(k / FEW_BUFS & 1));
      const int live = s_live[buf][warp];
      const bool draft = has_drafts && j == seg - 1;
      if (live > 0) {   // warp-uniform
        const unsigned kt = base + buf * FEW_STAGE, vt = kt + FEW_STAGE / 2;
        if (live < 16 || draft) {
          // A weight of zero does not keep out of the product what is not a number: rows that are not seen become zero, and so do a draft's
          // infinities and NaN, which the queries that see it get back at the end.
          for (int i = lane; i < 256; i += 32) {
            const int r = 16 * warp + (i >> 4);
            const unsigned at = vt + (i >> 3 & 1) * (FEW_STAGE / 4) + r * 128 + (i & 7) * 16;
            if (r - 16 * warp >= live) {
              asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(at), "r"(0) : "memory");
            } else if (draft) {
              uint32_t v[4];
              asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(at) : "memory");
              bool bad = false;
#pragma unroll
              for (int e = 0; e < 4; e++) bad |= not_finite(v[e]) | not_finite(v[e] >> 16);
              if (bad) {
                atomicOr(&s_bad, 1u << r);
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] = (not_finite(v[e]) ? 0 : v[e] & 0xffffu) | (not_finite(v[e] >> 16) ? 0 : v[e] & 0xffff0000u);
                asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
              }
            }
          }
          fence_async();   // before the copy that will fill the stage again
          __syncwarp();
        }
        float sc[2][4];
#pragma unroll
        for (int nt = 0; nt < 2; nt++) {
          float acc[2][4] = {};
          const int key = 16 * warp + 8 * nt + (lane & 7);
#pragma unroll
          for (int q = 0; q < 4; q++) {   // 32 channels each
            uint32_t b[4];
            ldmatrix4(b, kt + (q >> 1) * (FEW_STAGE / 4) + key * 128 + ((((q & 1) * 4 + (lane >> 3)) ^ (lane & 7)) << 4));
#pragma unroll
            for (int e = 0; e < 2; e++)
              mma16816(acc[e], qa[2 * q + e][0], PAIR ? 0u : qa[2 * q + e][RPT - 1], qa[2 * q + e][RPT], PAIR ? 0u : qa[2 * q + e][2 * RPT - 1], b[2 * e], b[2 * e + 1]);
          }
#pragma unroll
          for (int i = 0; i < 4; i++) sc[nt][i] = acc[0][i] + acc[1][i];
        }
        uint32_t pa[4];
#pragma unroll
        for (int e = 0; e < RPT; e++) {
          const uint32_t bits = draft ? s_mask[min((8 * e + g) / p.a.G, p.a.T - 1)] : live >= 16 ? ~0u : ((1u << live) - 1) << (16 * (warp & 1));
          float x[4], mx = -INFINITY;
#pragma unroll
          for (int i = 0; i < 4; i++) {   // n-tile i / 2, column 2 t4 + i % 2
            const int key = 16 * (warp & 1) + 8 * (i >> 1) + 2 * t4 + (i & 1);
            x[i] = bits >> key & 1 && (!draft || warp < 2) ? sc[i >> 1][2 * e + (i & 1)] : -INFINITY;
            mx = fmaxf(mx, x[i]);
          }
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          const float m_new = fmaxf(m[e], mx), least = m_new == -INFINITY ? 0.0f : m_new;
          const float f = m_new > m[e] ? ex2((m[e] - m_new) * scale) : 1.0f;
          float y[4], sum = 0.0f;
#pragma unroll
          for (int i = 0; i < 4; i++) y[i] = ex2((x[i] - least) * scale), sum += y[i];
          l[e] = l[e] * f + sum, m[e] = m_new;
          if (__any_sync(0xffffffffu, f != 1.0f)) {
#pragma unroll
            for (int n = 0; n < 16; n++) {
              o[n][2 * e] *= f, o[n][2 * e + 1] *= f;
              if (PAIR) o[n][2] *= f, o[n][3] *= f;
            }
          }
#pragma unroll
          for (int nt = 0; nt < 2; nt++) {
            const uint32_t hi = pack2(y[2 * nt], y[2 * nt + 1]);
            pa[2 * nt + e] = hi;
            if (PAIR) pa[2 * nt + 1] = pack2(y[2 * nt] - __uint_as_float(hi << 16), y[2 * nt + 1] - __uint_as_float(hi & 0xffff0000u));
          }
        }
        const int vkey = 16 * warp + (lane >> 3 & 1) * 8 + (lane & 7);
#pragma unroll
        for (int np = 0; np < 8; np++) {
          uint32_t b[4];
          ldmatrix4t(b, vt + (np >> 2) * (FEW_STAGE / 4) + vkey * 128 + ((((np & 3) * 2 + (lane >> 4)) ^ (lane & 7)) << 4));
          mma16816(o[2 * np], pa[0], pa[1], pa[2], pa[3], b[0], b[1]);
          mma16816(o[2 * np + 1], pa[0], pa[1], pa[2], pa[3], b[2], b[3]);
        }
      }
      __syncwarp();
      if (j < seg - 1 && lane == 0) mbar_arrive1(empty + 8 * buf);   // (the stage of the segment's last tile first serves the warps' partials)
    }
    // ---- the four warps' shares of the segment ----
    float* s_o = reinterpret_cast<float*>(dyn + (base - smem_addr(dyn)) + (k - 1) % FEW_BUFS * FEW_STAGE);   // [4][8][FEW_OS]
#pragma unroll
    for (int e = 0; e < RPT; e++) {
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
      if (t4 == 0) s_m[warp][8 * e + g] = m[e] * scale, s_l[warp][8 * e + g] = l[e];
    }
    named_barrier(1, 128);
    const uint32_t bad = has_drafts ? s_bad : 0;
    float* rec = whole ? nullptr : p.records + (2 * (int64_t)blockIdx.x + (seg_first == 0)) * (ROWS * 130);
#pragma unroll
    for (int round = 0; round < ROWS / 8; round++) {
      if (8 * round < n_rows) {
        const int r = 8 * round + g;
        const float M = fmaxf(fmaxf(s_m[0][r], s_m[1][r]), fmaxf(s_m[2][r], s_m[3][r]));
        const float f = s_m[warp][r] == -INFINITY ? 0.0f : ex2(s_m[warp][r] - M);
        const int e = PAIR ? 0 : round;
        float* to = s_o + (warp * 8 + g) * FEW_OS + 2 * t4;
#pragma unroll
        for (int n = 0; n < 16; n++) {
          float2 v = make_float2(o[n][2 * e], o[n][2 * e + 1]);
          // an infinite value times what a rounding left is an infinity of any sign, or NaN where nothing was left: the other half has it
          if (PAIR) v.x += finite(o[n][2]) ? o[n][2] : 0.0f, v.y += finite(o[n][3]) ? o[n][3] : 0.0f;
          *reinterpret_cast<float2*>(to + 8 * n) = make_float2(v.x * f, v.y * f);
        }
        named_barrier(1, 128);
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const int row = 8 * round + i;
          if (row < n_rows) {
            const float Mi = fmaxf(fmaxf(s_m[0][row], s_m[1][row]), fmaxf(s_m[2][row], s_m[3][row]));
            float L = 0.0f, O = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; w++) {
              L += s_l[w][row] * (s_m[w][row] == -INFINITY ? 0.0f : ex2(s_m[w][row] - Mi));   // (a NaN stays: all scores that a warp saw were NaN)
              O += s_o[(w * 8 + i) * FEW_OS + tid];
            }
            if (s_dead) L = NAN;
            const int t = row_token(row), hq = row_head(row);
            if (bad)
              for (uint32_t left = bad & s_mask[t]; left; left &= left - 1) {
                const uint16_t v = p.a.dv[cur.b * p.a.dv_b + (int64_t)(__ffs(left) - 1) * p.a.dv_t + cur.h * p.a.dv_h + tid];
                if (not_finite(v)) O += bf2f(v);
              }
            if (whole) {
              const int64_t out_row = ((int64_t)cur.b * p.a.T + t) * Hq + hq;
              p.a.out[out_row * 128 + tid] = f2bf(L == 0.0f ? 0.0f : O / L);
              if (p.a.lse && tid == 0) p.a.lse[out_row] = L == 0.0f ? -INFINITY : Mi + log2f(L);
            } else {
              rec[row * 128 + tid] = O;
              if (tid == 0) rec[ROWS * 128 + row] = Mi, rec[ROWS * 129 + row] = L;
            }
          }
        }
        named_barrier(1, 128);
      }
    }
    if (has_drafts && tid == 0) s_bad = 0;
    fence_async();
    __syncwarp();
    if (lane == 0) mbar_arrive1(empty + 8 * ((k - 1) % FEW_BUFS));
    if (TREE) named_barrier(1, 128);   // the marks are clear
    for (int j = 0; j < seg; j++) cur.step(p);
  }
}

// A block per query row: the records of the blocks that share its item, in the order of the tiles.
template <bool TREE, int ROWS>
__global__ void __launch_bounds__(128) few_merge_kernel(const __grid_constant__ FewParams p, int blocks) {
  pdl_wait();
  pdl_trigger();
  __shared__ MergeShared shared;
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x & 31, Hq = p.a.H * p.a.G, hq = (int)(row % Hq), h = hq / p.a.G, g = hq % p.a.G;
  const int64_t bt = row / Hq;
  const int t = (int)(bt % p.a.T), b = (int)(bt / p.a.T), r = TREE ? t * p.a.G + g : g % ROWS;
  int64_t total = 0, first;
  int n;
  if (TREE) {
    int64_t before = 0;
    for (int b0 = 0; b0 < p.bs; b0 += 32) {
      const int tiles = b0 + lane < p.bs ? few_tiles(p, b0 + lane) : 0;
      total += (int64_t)p.a.H * __reduce_add_sync(0xffffffffu, tiles), before += (int64_t)p.a.H * __reduce_add_sync(0xffffffffu, b0 + lane < b ? tiles : 0);
    }
    n = few_tiles(p, b);
    first = before + (int64_t)h * n;
  } else {
    n = p.tiles, total = (int64_t)p.bs * p.a.T * p.a.H * p.row_groups * n;
    first = ((bt * p.a.H + h) * p.row_groups + g / ROWS) * n;
  }
  const unsigned shares = (unsigned)min((int64_t)blocks, total);
  const int c0 = share_owner(first, total, shares), c1 = share_owner(first + n - 1, total, shares);
  if (c0 == c1) return;   // written by its block
  merge_row(shared, c1 - c0 + 1, ROWS, r, [&](int i) { return p.records + (2 * (int64_t)(c0 + i) + (i == 0)) * (ROWS * 130); }, p.a.out + row * 128, p.a.lse ? p.a.lse + row : nullptr);
}

template <bool TREE, int ROWS>
int launch(const FewParams& p, const CUtensorMap (&maps)[4], int64_t most, const char* what, cudaStream_t st) {
  const int64_t slots = (int64_t)FEW_CTAS * sm_count();
  const int blocks = (int)(most < slots ? most : slots);
  static PerDevice opted;
  if (const unsigned long long bit = first_on_device(opted)) {
    if (cudaFuncSetAttribute(attend_few_kernel<TREE, ROWS>, cudaFuncAttributeMaxDynamicSharedMemorySize, FEW_SMEM) != cudaSuccess)
      return fail(PK_ERR_CUDA, "%s: %s", what, cudaGetErrorString(cudaGetLastError()));
    mark_on_device(opted, bit);
  }
  StageTimer timer(ST_ATTENTION, st);
  launch_chain(attend_few_kernel<TREE, ROWS>, dim3((unsigned)blocks), dim3(FEW_THREADS), FEW_SMEM, st, maps[0], maps[1], maps[2], maps[3], p);
  const int64_t rows = (int64_t)p.bs * p.a.T * p.a.H * p.a.G;
  launch_chain(few_merge_kernel<TREE, ROWS>, dim3((unsigned)rows), dim3(128), 0, st, p, blocks);
  return check_launch(what, 2);
}

}  // namespace

int64_t attend_few_workspace() { return 2 * (int64_t)FEW_CTAS * sm_count() * 16 * 130 * 4; }

int launch_attend_few(const AttendParams& a, int64_t bs, void* workspace, const char* what, cudaStream_t st) {
  const bool tree = a.blocks == nullptr;
  FewParams p = {};
  p.a = a, p.bs = (int)bs, p.records = (float*)workspace;
  const int rows = tree ? a.T * a.G : a.G, per = rows <= 8 ? 8 : 16;
  p.row_groups = tree ? 1 : (a.G + per - 1) / per;
  p.box = tree ? FEW_TILE : a.block < FEW_TILE ? a.block : FEW_TILE;
  p.tiles = tree ? 0 : (int)(((int64_t)a.n * a.block + FEW_TILE - 1) / FEW_TILE);
  CUtensorMap maps[4];
  bool ok = rows_map(&maps[0], a.k, a.cap, a.k_l, a.H, a.k_h, bs, a.k_b, p.box) && rows_map(&maps[1], a.v, a.cap, a.v_l, a.H, a.v_h, bs, a.v_b, p.box);
  if (tree) ok = ok && rows_map(&maps[2], a.dk, a.T, a.dk_t, a.H, a.dk_h, bs, a.dk_b, 32) && rows_map(&maps[3], a.dv, a.T, a.dv_t, a.H, a.dv_h, bs, a.dv_b, 32);
  else maps[2] = maps[0], maps[3] = maps[1];
  if (!ok) return launch_attend_rows(a, bs, what, st);
  const int64_t most = tree ? bs * a.H * ((a.cap + FEW_TILE - 1) / FEW_TILE + 1) : bs * a.T * a.H * p.row_groups * (int64_t)p.tiles;
  if (tree) return per == 8 ? launch<true, 8>(p, maps, most, what, st) : launch<true, 16>(p, maps, most, what, st);
  return per == 8 ? launch<false, 8>(p, maps, most, what, st) : launch<false, 16>(p, maps, most, what, st);
}

}  // namespace pk
