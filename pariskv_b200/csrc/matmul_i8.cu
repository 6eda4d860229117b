// Product of tokens and a matrix in 8-bit whole numbers:  out[t,o] = bf16( (sum_k x[t,k] w[o,k]) sx[t] so[o] ),  the sum in 32-bit whole numbers, exact.
//
// Up to four tokens: the matrix' bytes bound it, and dp4a on rows in registers is enough (matvec_i8_kernel).
// More: tcgen05.mma (kind::i8), 128 rows of the matrix are the 128 lanes of tensor memory, NT tokens its columns; 128 columns of both operands a stage, by TMA.  Where there are few tiles a cluster of blocks shares a
// tile's columns, so that all SMs copy, and their partial sums meet through distributed shared memory (matmul_i8_kernel).
// Many tokens: the tensor cores bound it.  Pairs of SMs share tiles of 256 x 256 and go from one to the next, the sums of one leave tensor memory under the products of the next (matmul_i8_pair_kernel).
// B200: 2048 tokens, 24576 x 4096 in 130 us, 3160 TOP/s, tensor cores busy 91 % of the time; 206 us with single SMs on tiles of 128 x 256 and a store loop whose reads the compiler had to keep behind its stores, 192 with
// pairs, 130 with the tokens' scales in shared memory and sixteen sums scaled before the first is stored.
#include "cache8.cuh"
#include "tiles.cuh"

namespace pk {
namespace {

constexpr int MM_THREADS = 320;        // a warp for the copies, one for the products, eight that scale and store: two for every quarter of the rows, each with half of the tokens
constexpr int MM_ROWS = 128, MM_K = 128;
constexpr int MM_WAIT_LIMIT = 100000;  // tries; one waits up to 10 us by itself

struct MmParams {
  const float *sx, *so;
  uint16_t* out;
  int64_t out_t;      // stride of a token's row
  int T, O, chunks;   // chunks of 128 columns
  int t_tiles, tiles; // tiles of tokens; tiles in all, tokens first
  int split;          // blocks of a cluster
};

// Two blocks per SM: the start and the end of one lie under the copies of the other.
template <int NT> struct MmRing {
  static constexpr int bytes = MM_ROWS * MM_K + NT * MM_K, ctas = 2, stages = NT >= 128 ? 3 : NT >= 64 ? 4 : 5;
};
template <int NT> constexpr int mm_smem() { return 1024 + MmRing<NT>::stages * MmRing<NT>::bytes; }

__device__ __forceinline__ void tma_load2(unsigned dst, const CUtensorMap* map, int c0, int c1, unsigned mb) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(mb) : "memory");
}
// D[tmem] (+)= A[smem] B[smem]: 8-bit whole numbers, 32-bit sums
__device__ __forceinline__ void tc_mma_i8(unsigned d, uint64_t a, uint64_t b, unsigned idesc, unsigned add) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(add) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t (&r)[16], unsigned addr) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
                 "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void tmem_wait16(uint32_t (&r)[16]) {   // the values are there behind it, and no use of them moves before it
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]),
                 "+r"(r[14]), "+r"(r[15])::"memory");
}
// A lane's row of sums - matrix row o, the tile's tokens c0 .. c1, t0 the first of the tile - out of tensor memory, scaled and stored; sx: the tokens' scales.  The next sixteen are under way while sixteen
// are stored; all of a step's reads come before its stores, which the compiler must not reorder.
template <class Free>
__device__ __forceinline__ void mm_store(const MmParams& p, unsigned addr, int c0, int c1, int t0, int o, const float* sx, bool dead, Free all_read) {
  const float so = o < p.O ? p.so[o] : 0.0f;
  uint16_t* to = p.out + (t0 + c0) * p.out_t + o;
  const bool inside = t0 + c1 <= p.T;
  uint32_t next[16];
  if (c0 < c1) tmem_ld16(next, addr + c0);
#pragma unroll 1
  for (int c = c0; c < c1; c += 16) {
    uint32_t acc[16];
    tmem_wait16(next);
#pragma unroll
    for (int i = 0; i < 16; i++) acc[i] = next[i];
    if (c + 16 < c1) tmem_ld16(next, addr + c + 16);
    else all_read();
    uint16_t y[16];
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const float4 s = *reinterpret_cast<const float4*>(sx + c + i);
      y[i] = f2bf((float)(int)acc[i] * s.x * so), y[i + 1] = f2bf((float)(int)acc[i + 1] * s.y * so);
      y[i + 2] = f2bf((float)(int)acc[i + 2] * s.z * so), y[i + 3] = f2bf((float)(int)acc[i + 3] * s.w * so);
    }
    if (dead) {
#pragma unroll
      for (int i = 0; i < 16; i++) y[i] = 0x7fff;
    }
    if (o < p.O) {
#pragma unroll
      for (int i = 0; i < 16; i++, to += p.out_t)
        if (inside || t0 + c + i < p.T) *to = y[i];
    }
  }
  if (c0 >= c1) all_read();
}
__device__ __forceinline__ void cluster_sync() { asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint4 remote16(unsigned at, unsigned rank) {   // the same place in the shared memory of block `rank` of the cluster
  uint4 r;
  asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %4, %5;\n\tld.shared::cluster.v4.b32 {%0,%1,%2,%3}, [a];\n\t}" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(at), "r"(rank) : "memory");
  return r;
}
__device__ __forceinline__ unsigned remote4(unsigned at, unsigned rank) {
  unsigned r;
  asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %1, %2;\n\tld.shared::cluster.u32 %0, [a];\n\t}" : "=r"(r) : "r"(at), "r"(rank) : "memory");
  return r;
}

template <int NT>
__global__ void __launch_bounds__(MM_THREADS, MmRing<NT>::ctas) matmul_i8_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ MmParams p) {
  constexpr int NS = MmRing<NT>::stages, STAGE = MmRing<NT>::bytes, COLS = NT < 32 ? 32 : NT;   // columns of a set of sums
  constexpr unsigned IDESC = 2u << 4 | 1u << 7 | 1u << 10 | (unsigned)(NT >> 3) << 17 | (unsigned)(MM_ROWS >> 4) << 24;
  extern __shared__ unsigned char dyn[];
  __shared__ __align__(8) unsigned long long bars[2 * NS + 5];
  __shared__ unsigned s_tmem;
  __shared__ __align__(16) float s_sx[2][NT];
  __shared__ __align__(16) volatile int s_dead;
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const unsigned ring = (smem_addr(dyn) + 1023) & ~1023u;
  const unsigned full = smem_addr(bars), empty = full + 8 * NS, done = empty + 8 * NS, taken = done + 16, ending = taken + 16;
  if (tid == 0) {
    for (int i = 0; i < NS; i++) mbar_init(full + 8 * i, 1), mbar_init(empty + 8 * i, 1);
    for (int i = 0; i < 2; i++) mbar_init(done + 8 * i, 1), mbar_init(taken + 8 * i, 256);
    mbar_init(ending, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    s_dead = 0;
  }
  if (warp == 1) tmem_alloc(smem_addr(&s_tmem), 2 * COLS);
  if (warp == 0 && lane < 2) tma_prefetch_map(lane ? &map_x : &map_w);
  const int rank = (int)(blockIdx.x % p.split), cluster = (int)(blockIdx.x / p.split), clusters = (int)(gridDim.x / p.split);
  const int k0 = (int)((int64_t)p.chunks * rank / p.split), k1 = (int)((int64_t)p.chunks * (rank + 1) / p.split);
  if (warp == 0 && lane == 0)   // the first columns on their way to L2 while the kernel before ends: 16 x 6144 x 4096 8.0 -> 7.7 us, 128 x 6144 x 4096 12.0 -> 11.6
    for (int k = k0; k < min(k1, k0 + NS); k++)
      asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(&map_w), "r"(k * MM_K), "r"(cluster / p.t_tiles * MM_ROWS) : "memory");
  pdl_wait();
  pdl_trigger();
  tc_before();
  __syncthreads();
  tc_after();
  const unsigned tmem = s_tmem;
  bool dead = false;   // a wait has run out: no more waiting, the sums come out as NaN
  auto wait = [&](unsigned mb, unsigned parity) {
    for (int it = 0; !dead; it++) {
      if (mbar_try(mb, parity)) break;
      if (it >= MM_WAIT_LIMIT || ((it & 1023) == 1023 && s_dead)) dead = true, s_dead = 1;
    }
  };
  if (warp == 0) {
    if (lane == 0) {
      int q = 0;
      for (int tile = cluster; tile < p.tiles && !dead; tile += clusters) {
        const int t0 = tile % p.t_tiles * NT, o0 = tile / p.t_tiles * MM_ROWS;
        for (int k = k0; k < k1; k++, q++) {
          const int st = q % NS;
          if (q >= NS) wait(empty + 8 * st, (unsigned)(q / NS - 1) & 1);
          if (dead) break;
          mbar_expect(full + 8 * st, STAGE);
          tma_load2(ring + st * STAGE, &map_w, k * MM_K, o0, full + 8 * st);
          tma_load2(ring + st * STAGE + MM_ROWS * MM_K, &map_x, k * MM_K, t0, full + 8 * st);
        }
      }
      if (dead || s_dead)   // what is under way has to land before the block ends
        for (int i = q < NS ? 0 : q - NS; i < q; i++)
          for (int it = 0; it < MM_WAIT_LIMIT && !mbar_try(full + 8 * (i % NS), (unsigned)(i / NS) & 1); it++) {}
    }
  } else if (warp == 1) {
    const bool leader = elect_one();
    const uint64_t w_desc = umma_desc(ring, 16), x_desc = umma_desc(ring + MM_ROWS * MM_K, 16);
    int q = 0, n = 0;
    for (int tile = cluster; tile < p.tiles; tile += clusters, n++) {
      const int set = n & 1;
      if (n >= 2) wait(taken + 8 * set, (unsigned)(n / 2 - 1) & 1);
      __syncwarp();
      tc_after();
      for (int k = k0; k < k1; k++, q++) {
        const int st = q % NS;
        wait(full + 8 * st, (unsigned)(q / NS) & 1);
        __syncwarp();
        tc_after();
        if (leader && !dead) {
          const uint64_t a = w_desc + (uint64_t)st * (STAGE >> 4), b = x_desc + (uint64_t)st * (STAGE >> 4);
#pragma unroll
          for (int i = 0; i < 4; i++) tc_mma_i8(tmem + COLS * set, a + 2 * i, b + 2 * i, IDESC, k > k0 || i > 0);
          tc_commit(empty + 8 * st);
        }
      }
      if (leader && !dead) tc_commit(done + 8 * set);
    }
    if (s_dead && leader) {   // products under way end before the tensor memory goes
      tc_commit(ending);
      for (int it = 0; it < MM_WAIT_LIMIT && !mbar_try(ending, 0); it++) {}
    }
  } else {
    const int quarter = warp & 3, o_lane = 32 * quarter + lane, part = (warp - 2) >> 2, c0 = NT >= 32 ? part * (NT / 2) : part * NT, c1 = NT >= 32 ? c0 + NT / 2 : NT;
    const unsigned lanes = tmem + ((unsigned)quarter << 21);
    int n = 0;
    for (int tile = cluster; tile < p.tiles; tile += clusters, n++) {
      const int set = n & 1, t0 = tile % p.t_tiles * NT, o = tile / p.t_tiles * MM_ROWS + o_lane;
      if (p.split == 1) {   // (the threads before the ones of this tile have passed the barrier of the tile before: two places do)
        for (int i = tid - 64; i < NT; i += 256) s_sx[set][i] = t0 + i < p.T ? p.sx[t0 + i] : 0.0f;
        named_barrier(1, 256);
      }
      wait(done + 8 * set, (unsigned)(n / 2) & 1);
      __syncwarp();
      tc_after();
      if (p.split == 1) {
        mm_store(p, lanes + COLS * set, c0, c1, t0, o, s_sx[set], dead, [&] {
          tc_before();
          mbar_arrive1(taken + 8 * set);
        });
      } else {
        // this block's partial sums, column by column, where the copies were (they have all been multiplied)
#pragma unroll 1
        for (int c = c0; c < c1; c += 16) {
          uint32_t acc[16];
          tmem_ld16(acc, lanes + COLS * set + c);
          tmem_wait16(acc);
#pragma unroll
          for (int i = 0; i < 16; i++) asm volatile("st.shared.b32 [%0], %1;" ::"r"(ring + ((c + i) * MM_ROWS + o_lane) * 4), "r"(acc[i]) : "memory");
        }
      }
    }
  }
  if (p.split > 1) {   // one tile a cluster.  Column t of the tile, four rows a thread: the block that has t mod split adds them
    __syncwarp();
    tc_before();
    cluster_sync();
    const int tile = cluster, t0 = tile % p.t_tiles * NT, o0 = tile / p.t_tiles * MM_ROWS;
    bool lost = false;
    for (int s = 0; s < p.split; s++) lost |= remote4(smem_addr((const void*)&s_dead), (unsigned)s) != 0;
    for (int c = rank * (MM_THREADS / 32) + warp; c < NT; c += p.split * (MM_THREADS / 32)) {
      const int t = t0 + c;
      if (t >= p.T) continue;
      uint4 sum = make_uint4(0, 0, 0, 0);
#pragma unroll 4
      for (int s = 0; s < p.split; s++) {
        const uint4 v = remote16(ring + (c * MM_ROWS + 4 * lane) * 4, (unsigned)s);
        sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
      }
      const uint32_t a[4] = {sum.x, sum.y, sum.z, sum.w};
      const float sx = p.sx[t];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int o = o0 + 4 * lane + i;
        if (o < p.O) p.out[t * p.out_t + o] = f2bf(lost ? NAN : (float)(int)a[i] * sx * p.so[o]);
      }
    }
    cluster_sync();
  }
  tc_before();
  __syncthreads();
  tc_after();
  if (warp == 1) tmem_free(tmem, 2 * COLS);
}

// ---- many tokens: two SMs on a tile of 256 rows and 256 tokens ----
// Each block of a pair copies 128 rows of the matrix and 128 tokens, and has the sums of its rows; a product reads both blocks' operands (cta_group::2), so that a block copies 32 KB for the work that takes 48 KB alone.
// The first block issues; copies of both arrive on its barriers, and its commits reach both.
constexpr int MP_NT = 256, MP_STAGES = 6, MP_STAGE = 2 * 128 * MM_K, MP_SMEM = 1024 + MP_STAGES * MP_STAGE;

__device__ __forceinline__ unsigned in_block0(unsigned at) {   // the same place in the pair's first block
  unsigned r;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(at));
  return r;
}
__device__ __forceinline__ void tma_load2_pair(unsigned dst, const CUtensorMap* map, int c0, int c1, unsigned mb) {   // mb: in either block of the pair
  asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(mb)
               : "memory");
}
__device__ __forceinline__ void tc_mma_i8_pair(unsigned d, uint64_t a, uint64_t b, unsigned idesc, unsigned add) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(add) : "memory");
}
__device__ __forceinline__ void tc_commit_pair(unsigned mb) {   // to that place of both blocks
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(mb), "h"((uint16_t)3) : "memory");
}

__global__ void __launch_bounds__(MM_THREADS, 1) matmul_i8_pair_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ MmParams p) {
  constexpr int NS = MP_STAGES, STAGE = MP_STAGE, NT = MP_NT;
  constexpr unsigned IDESC = 2u << 4 | 1u << 7 | 1u << 10 | (unsigned)(NT >> 3) << 17 | (unsigned)(256 >> 4) << 24;
  extern __shared__ unsigned char dyn[];
  __shared__ __align__(8) unsigned long long bars[2 * NS + 5];
  __shared__ unsigned s_tmem;
  __shared__ __align__(16) float s_sx[2][NT];
  __shared__ volatile int s_dead;
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const unsigned ring = (smem_addr(dyn) + 1023) & ~1023u;
  const unsigned full = smem_addr(bars), empty = full + 8 * NS, done = empty + 8 * NS, taken = done + 16, ending = taken + 16;
  const int rank = (int)(blockIdx.x & 1), pair = (int)(blockIdx.x >> 1), pairs = (int)(gridDim.x >> 1);
  if (tid == 0) {
    for (int i = 0; i < NS; i++) mbar_init(full + 8 * i, 1), mbar_init(empty + 8 * i, 1);
    for (int i = 0; i < 2; i++) mbar_init(done + 8 * i, 1), mbar_init(taken + 8 * i, 16);
    mbar_init(ending, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    s_dead = 0;
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&s_tmem)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  if (warp == 0 && lane < 2) tma_prefetch_map(lane ? &map_x : &map_w);
  pdl_wait();
  pdl_trigger();
  tc_before();
  __syncthreads();
  cluster_sync();   // the barriers of both are there
  tc_after();
  const unsigned tmem = s_tmem;
  bool dead = false;   // a wait has run out: no more waiting, the sums come out as NaN
  auto wait = [&](unsigned mb, unsigned parity) {
    for (int it = 0; !dead; it++) {
      if (mbar_try(mb, parity)) break;
      if (it >= MM_WAIT_LIMIT || ((it & 1023) == 1023 && s_dead)) dead = true, s_dead = 1;
    }
  };
  if (warp == 0) {
    if (lane == 0) {
      int q = 0;
      const unsigned full0 = in_block0(full);
      for (int tile = pair; tile < p.tiles && !dead; tile += pairs) {
        const int t0 = tile % p.t_tiles * NT + 128 * rank, o0 = tile / p.t_tiles * 256 + 128 * rank;
        for (int k = 0; k < p.chunks; k++, q++) {
          const int st = q % NS;
          if (q >= NS) wait(empty + 8 * st, (unsigned)(q / NS - 1) & 1);
          if (dead) break;
          if (rank == 0) mbar_expect(full + 8 * st, 2 * STAGE);
          tma_load2_pair(ring + st * STAGE, &map_w, k * MM_K, o0, full0 + 8 * st);
          tma_load2_pair(ring + st * STAGE + 128 * MM_K, &map_x, k * MM_K, t0, full0 + 8 * st);
        }
      }
      if (rank == 0 && (dead || s_dead))   // what is under way has to land before the blocks end
        for (int i = q < NS ? 0 : q - NS; i < q; i++)
          for (int it = 0; it < MM_WAIT_LIMIT && !mbar_try(full + 8 * (i % NS), (unsigned)(i / NS) & 1); it++) {}
    }
  } else if (warp == 1) {
    if (rank == 0) {
      const bool leader = elect_one();
      const uint64_t w_desc = umma_desc(ring, 16), x_desc = umma_desc(ring + 128 * MM_K, 16);
      int q = 0, n = 0;
      for (int tile = pair; tile < p.tiles; tile += pairs, n++) {
        const int set = n & 1;
        if (n >= 2) wait(taken + 8 * set, (unsigned)(n / 2 - 1) & 1);
        __syncwarp();
        tc_after();
        for (int k = 0; k < p.chunks; k++, q++) {
          const int st = q % NS;
          wait(full + 8 * st, (unsigned)(q / NS) & 1);
          __syncwarp();
          tc_after();
          if (leader && !dead) {
            const uint64_t a = w_desc + (uint64_t)st * (STAGE >> 4), b = x_desc + (uint64_t)st * (STAGE >> 4);
#pragma unroll
            for (int i = 0; i < 4; i++) tc_mma_i8_pair(tmem + NT * set, a + 2 * i, b + 2 * i, IDESC, k > 0 || i > 0);
            tc_commit_pair(empty + 8 * st);
          }
        }
        if (leader && !dead) tc_commit_pair(done + 8 * set);
      }
      if (s_dead && leader) {   // products under way end before the tensor memory goes
        tc_commit_pair(ending);
        for (int it = 0; it < MM_WAIT_LIMIT && !mbar_try(ending, 0); it++) {}
      }
    }
  } else {
    const int quarter = warp & 3, c0 = (warp - 2) / 4 * (NT / 2);
    const unsigned lanes = tmem + ((unsigned)quarter << 21), taken0 = in_block0(taken);
    int n = 0;
    for (int tile = pair; tile < p.tiles; tile += pairs, n++) {
      const int set = n & 1, t0 = tile % p.t_tiles * NT, o = tile / p.t_tiles * 256 + 128 * rank + 32 * quarter + lane;
      for (int i = tid - 64; i < NT; i += 256) s_sx[set][i] = t0 + i < p.T ? p.sx[t0 + i] : 0.0f;
      named_barrier(1, 256);
      wait(done + 8 * set, (unsigned)(n / 2) & 1);
      __syncwarp();
      tc_after();
      mm_store(p, lanes + NT * set, c0, c0 + NT / 2, t0, o, s_sx[set], dead, [&] {
        tc_before();
        __syncwarp();
        if (lane == 0) asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(taken0 + 8 * set) : "memory");
      });
    }
  }
  tc_before();
  __syncthreads();
  cluster_sync();   // neither block ends while the other may reach into it
  tc_after();
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
}

// ---- up to four tokens: no tensor cores ----
// Rows of the matrix straight into registers, 512 columns a warp and load, eight loads under way; four products an instruction (dp4a), a warp's sum in one (redux).  A block per SM has an even share of the
// rows; `cw` warps share a row's columns, with the tokens' values for them in registers, and add up in shared memory: whole numbers, so that the order does not matter.
constexpr int MV_THREADS = 512, MV_ROWS = 1024;   // rows between two stores
struct MvParams {
  const int8_t *w, *x;
  int64_t w_o, x_t;
  const float *sx, *so;
  uint16_t* out;
  int64_t out_t;
  int O, I, cw;
};
template <int T, int CH, int U>   // CH: loads of a row by a warp; U: rows at a time, and as many under way
__global__ void __launch_bounds__(MV_THREADS, 1) matvec_i8_kernel(const __grid_constant__ MvParams p) {
  __shared__ int s_sum[MV_ROWS * T];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int r0 = (int)((int64_t)p.O * blockIdx.x / gridDim.x), r1 = (int)((int64_t)p.O * (blockIdx.x + 1) / gridDim.x);
  const int groups = MV_THREADS / 32 / p.cw, group = warp / p.cw, col = (warp % p.cw) * 512 + lane * 16;
  if (lane == 0 && group < groups) {   // the first rows on their way to L2 while the kernel before ends
    for (int u = 0; u < U; u++)
      if (r0 + group * U + u < r1 && (warp % p.cw) * 512 < p.I)
        asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p.w + (int64_t)(r0 + group * U + u) * p.w_o + (warp % p.cw) * 512), "r"(min(512, p.I - (warp % p.cw) * 512)) : "memory");
  }
  pdl_wait();
  pdl_trigger();
  for (int i = tid; i < MV_ROWS * T; i += MV_THREADS) s_sum[i] = 0;
  int4 x[T][CH];
#pragma unroll
  for (int t = 0; t < T; t++)
#pragma unroll
    for (int c = 0; c < CH; c++)
      x[t][c] = col + c * p.cw * 512 < p.I ? *reinterpret_cast<const int4*>(p.x + t * p.x_t + col + c * p.cw * 512) : make_int4(0, 0, 0, 0);
  for (int base = r0; base < r1; base += MV_ROWS) {
    const int n = min(MV_ROWS, r1 - base);
    __syncthreads();
    if (group < groups) {
      int4 w[2][U][CH];
      auto load = [&](int4 (&to)[U][CH], int r) {
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
          for (int c = 0; c < CH; c++)
            to[u][c] = r + u < n && col + c * p.cw * 512 < p.I ? *reinterpret_cast<const int4*>(p.w + (int64_t)(base + r + u) * p.w_o + col + c * p.cw * 512) : make_int4(0, 0, 0, 0);
      };
      auto multiply = [&](const int4 (&w)[U][CH], int r) {
#pragma unroll
        for (int t = 0; t < T; t++) {
          int mine = 0;
#pragma unroll
          for (int u = 0; u < U; u++) {
            int a = 0;
#pragma unroll
            for (int c = 0; c < CH; c++)
              a = __dp4a(w[u][c].x, x[t][c].x, a), a = __dp4a(w[u][c].y, x[t][c].y, a), a = __dp4a(w[u][c].z, x[t][c].z, a), a = __dp4a(w[u][c].w, x[t][c].w, a);
            a = __reduce_add_sync(0xffffffffu, a);
            if (lane == u) mine = a;
          }
          if (lane < U && r + lane < n) atomicAdd(&s_sum[t * MV_ROWS + r + lane], mine);
        }
      };
      int r = group * U;
      load(w[0], r);
      for (; r < n; r += 2 * groups * U) {   // the next rows are under way
        load(w[1], r + groups * U);
        multiply(w[0], r);
        if (r + groups * U >= n) break;
        load(w[0], r + 2 * groups * U);
        multiply(w[1], r + groups * U);
      }
    }
    __syncthreads();
    for (int i = tid; i < n; i += MV_THREADS) {
      const float so = p.so[base + i];
#pragma unroll
      for (int t = 0; t < T; t++) {
        p.out[t * p.out_t + base + i] = f2bf((float)s_sum[t * MV_ROWS + i] * p.sx[t] * so);
        s_sum[t * MV_ROWS + i] = 0;
      }
    }
  }
}

template <int T, int CH, int U>
int launch_vec_as(const MvParams& p, int blocks, cudaStream_t st) {
  StageTimer timer(ST_GEMV, st);
  launch_chain(matvec_i8_kernel<T, CH, U>, dim3((unsigned)blocks), dim3(MV_THREADS), 0, st, p);
  return check_launch("matmul_i8");
}
// Rows at a time: four of 512 columns where a warp has few (B200, us, one token, one matrix again and again, four | eight at a time: 1024 x 1024 1.9 | 2.7, 6144 x 4096 4.3 | 5.3), eight where it has many (12288 x 4096 11.2 | 10.3,
// 24576 x 4096 18.9 | 17.5, 151936 x 4096 95 | 91).
template <int T>
int launch_vec(MvParams p, cudaStream_t st) {
  const int loads = (p.I + 511) / 512;
  p.cw = loads < 8 ? loads : 8;
  const int per = (loads + p.cw - 1) / p.cw, groups = MV_THREADS / 32 / p.cw, sms = sm_count(), most = (p.O + groups - 1) / groups, blocks = most < sms ? most : sms;
  const bool many = p.O / (blocks * groups) >= 32;
  if (per == 1) return many ? launch_vec_as<T, 1, 8>(p, blocks, st) : launch_vec_as<T, 1, 4>(p, blocks, st);
  if (per == 2) return many ? launch_vec_as<T, 2, 4>(p, blocks, st) : launch_vec_as<T, 2, 2>(p, blocks, st);
  if constexpr (T < 4)
    if (per == 4) return launch_vec_as<T, 4, 2>(p, blocks, st);
  return launch_vec_as<T, 3, 2>(p, blocks, st);
}
constexpr int MV_MOST = 4 * 8 * 512;   // columns

// Rows of 8-bit numbers in boxes of 128 columns; what is behind the last row or column comes as zeros.
bool bytes_map(CUtensorMap* m, const void* base, int64_t rows, int64_t cols, int64_t stride, int box) {
  const auto encode = tensor_map_encoder();
  if (!encode) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)stride};
  const cuuint32_t boxes[2] = {MM_K, (cuuint32_t)box}, steps[2] = {1, 1};
  return encode(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Blocks that share a tile's columns: as many as there are SMs for, each with so many steps that the sums' way through shared memory is worth it.  B200, us, 4096 columns (one matrix again and again), by 1 | 2 | 3 | 4 | 6 | 8 blocks:
// 16 tokens, 1024 rows 9.6 | 7.6 | 6.3 | 5.5 | 5.6 | 5.2, 6144 rows 10.4 | 8.3 | 7.6 | 7.6 | 12.0 | 11.6, 24576 rows 18.9 | 26 | 30 | 28 | 39 | 42;  128 tokens, 6144 rows 13.4 | 15.5 | 14.2 | 12.8 | 21 | 20.
int mm_split(int64_t tiles, int chunks, int nt) {
  const int least = nt / 8;
  int s = 1;
  while (s < 8 && tiles * (s + 1) <= sm_count() && chunks >= (s + 1) * least) s++;
  return s;
}

template <int NT>
int launch(const pk_tensor* x, const pk_tensor* w, MmParams p, cudaStream_t st) {
  CUtensorMap mw, mx;
  const int64_t I = x->shape[1];
  if (!bytes_map(&mw, w->data, p.O, I, p.O > 1 ? w->stride[0] : (I + 15) / 16 * 16, MM_ROWS) || !bytes_map(&mx, x->data, p.T, I, p.T > 1 ? x->stride[0] : (I + 15) / 16 * 16, NT))
    return fail(PK_ERR_CUDA, "matmul_i8: no tensor map for these rows");
  static PerDevice opted;
  if (const unsigned long long bit = first_on_device(opted)) {
    if (cudaFuncSetAttribute(matmul_i8_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, mm_smem<NT>()) != cudaSuccess)
      return fail(PK_ERR_CUDA, "matmul_i8: %s", cudaGetErrorString(cudaGetLastError()));
    mark_on_device(opted, bit);
  }
  p.t_tiles = (p.T + NT - 1) / NT;
  p.tiles = p.t_tiles * ((p.O + MM_ROWS - 1) / MM_ROWS);
  const int slots = MmRing<NT>::ctas * sm_count();
  p.split = mm_split(p.tiles, p.chunks, NT);
  const int clusters = p.split > 1 ? p.tiles : p.tiles < slots ? p.tiles : slots;
  StageTimer timer(ST_GEMV, st);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(clusters * p.split)), cfg.blockDim = dim3(MM_THREADS), cfg.dynamicSmemBytes = mm_smem<NT>(), cfg.stream = st;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (p.split > 1) attr[n].id = cudaLaunchAttributeClusterDimension, attr[n].val.clusterDim.x = (unsigned)p.split, attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1, n++;
  if (pdl_enabled()) attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization, attr[n].val.programmaticStreamSerializationAllowed = 1, n++;
  cfg.attrs = attr, cfg.numAttrs = n;
  cudaLaunchKernelEx(&cfg, matmul_i8_kernel<NT>, mw, mx, p);
  return check_launch("matmul_i8");
}

int launch_pair(const pk_tensor* x, const pk_tensor* w, MmParams p, cudaStream_t st) {
  CUtensorMap mw, mx;
  const int64_t I = x->shape[1];
  if (!bytes_map(&mw, w->data, p.O, I, p.O > 1 ? w->stride[0] : I, 128) || !bytes_map(&mx, x->data, p.T, I, p.T > 1 ? x->stride[0] : I, 128))
    return fail(PK_ERR_CUDA, "matmul_i8: no tensor map for these rows");
  static PerDevice opted;
  if (const unsigned long long bit = first_on_device(opted)) {
    if (cudaFuncSetAttribute(matmul_i8_pair_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MP_SMEM) != cudaSuccess)
      return fail(PK_ERR_CUDA, "matmul_i8: %s", cudaGetErrorString(cudaGetLastError()));
    mark_on_device(opted, bit);
  }
  p.t_tiles = (p.T + MP_NT - 1) / MP_NT;
  p.tiles = p.t_tiles * ((p.O + 255) / 256);
  p.split = 1;
  const int pairs = sm_count() / 2;
  StageTimer timer(ST_GEMV, st);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * (p.tiles < pairs ? p.tiles : pairs))), cfg.blockDim = dim3(MM_THREADS), cfg.dynamicSmemBytes = MP_SMEM, cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension, attr[0].val.clusterDim.x = 2, attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization, attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr, cfg.numAttrs = pdl_enabled() ? 2 : 1;
  cudaLaunchKernelEx(&cfg, matmul_i8_pair_kernel, mw, mx, p);
  return check_launch("matmul_i8");
}

bool rows16(const pk_tensor* t) {
  return (t->shape[1] <= 1 || t->stride[1] == 1) && aligned16(t->data) && (t->shape[0] <= 1 || (t->stride[0] % 16 == 0 && t->stride[0] > 0));
}

}  // namespace
}  // namespace pk

using namespace pk;

extern "C" int pk_matmul_i8(const pk_tensor* x, const pk_tensor* x_scales, const pk_tensor* weight, const pk_tensor* weight_scales, const pk_tensor* out, void* stream) {
  PK_CHECK_TENSOR(x, PK_I8, 2);
  PK_CHECK_TENSOR(x_scales, PK_F32, 1);
  PK_CHECK_TENSOR(weight, PK_I8, 2);
  PK_CHECK_TENSOR(weight_scales, PK_F32, 1);
  PK_CHECK_TENSOR(out, PK_BF16, 2);
  const int64_t T = x->shape[0], I = x->shape[1], O = weight->shape[0];
  PK_REQUIRE(I >= 16 && I % 16 == 0 && I <= 65536, "the width must be a multiple of 16, at most 65536");
  PK_REQUIRE(weight->shape[1] == I, "weight must be i8 [O,I], as wide as x");
  PK_REQUIRE(T < (1LL << 31) - 256 && O < (1LL << 31) - 256 && ((T + 15) / 16) * ((O + 127) / 128) < (1LL << 31), "sizes out of range");
  PK_REQUIRE(rows16(x) && rows16(weight), "x and weight need a unit inner stride, rows at strides that are multiples of 16, and 16-byte alignment");
  PK_REQUIRE(x_scales->shape[0] == T && is_contig(x_scales), "x_scales must be contiguous f32 [T]");
  PK_REQUIRE(weight_scales->shape[0] == O && is_contig(weight_scales), "weight_scales must be contiguous f32 [O]");
  PK_REQUIRE(out->shape[0] == T && out->shape[1] == O && (O <= 1 || out->stride[1] == 1) && (T <= 1 || out->stride[0] >= O), "out must be bf16 [T,O] with a unit inner stride, rows apart");
  if (T == 0 || O == 0) return PK_OK;
  MmParams p = {};
  p.sx = (const float*)x_scales->data, p.so = (const float*)weight_scales->data, p.out = (uint16_t*)out->data, p.out_t = out->stride[0];
  p.T = (int)T, p.O = (int)O, p.chunks = (int)((I + MM_K - 1) / MM_K);
  const cudaStream_t st = (cudaStream_t)stream;
  // Which kernel, B200, us, without | with tensor cores, one matrix again and again (from L2): 6144 x 4096, one token 4.3 | 8.2, three 5.8 | 7.6, four 6.5 | 7.5; 24576 x 4096, two tokens 18.5 | 19.6, four 20.8 | 19.6;
  // 3000 x 16384, three tokens 8.1 | 10.0, but four, whose values and sums do not fit into the registers from 12289 columns on, 12.5 | 10.1.  Matrices of 300 MB in turn: 6144 x 4096, four tokens 8.1 | 9.2,
  // 4096 x 12288 10.8 | 12.9, 3000 x 16384 15.9 | 14.0.
  if (I <= MV_MOST && (T <= 2 || (T <= 4 && O * I <= 48 << 20 && (T == 3 || I <= MV_MOST * 3 / 4)))) {
    const MvParams v = {(const int8_t*)weight->data, (const int8_t*)x->data, O > 1 ? weight->stride[0] : I, T > 1 ? x->stride[0] : I, p.sx, p.so, p.out, p.out_t, (int)O, (int)I, 0};
    return T == 1 ? launch_vec<1>(v, st) : T == 2 ? launch_vec<2>(v, st) : T == 3 ? launch_vec<3>(v, st) : launch_vec<4>(v, st);
  }
  if (T <= 16) return launch<16>(x, weight, p, st);
  if (T <= 32) return launch<32>(x, weight, p, st);
  if (T <= 64) return launch<64>(x, weight, p, st);
  // Tiles of 128 rows and 64 tokens, two blocks an SM, or of 256 x 256 on pairs, by what a round of each takes: 0.33 or 0.4 us for 128 columns, at least 0.6 or 2.3 us for its sums' way out.
  // 256 x 6144 x 4096 13.5 | 16.2, 512 x 4096 x 12288 32 | 34, 512 x 6144 x 4096 21.8 | 17.4, 2048 x 4096 x 12288 109 | 65, 533 x 17888 x 96 11.5 | 14.1.
  const int64_t small = (T + 63) / 64 * ((O + 127) / 128), large = (T + 255) / 256 * ((O + 255) / 256), small_places = 2 * sm_count(), pairs = sm_count() / 2;
  const int64_t small_round = 33 * p.chunks > 60 ? 33 * p.chunks : 60, large_round = 40 * p.chunks > 230 ? 40 * p.chunks : 230;
  if (small <= small_places || (T > 128 && (small + small_places - 1) / small_places * small_round < (large + pairs - 1) / pairs * large_round)) return launch<64>(x, weight, p, st);
  if (T <= 128) return launch<128>(x, weight, p, st);
  return launch_pair(x, weight, p, st);
}
