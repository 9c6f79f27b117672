// Ragged products by group on the tcgen05 tensor cores: y = x w_g^T, dx = dy w_g, dw_g = dy_g^T x_g in
// 16 bits, and y = a b_g^T of microscaled rows (e2m1 or e4m3 with a power of two for 32 values).
//
// All of them are D[128][BN] += P Q^T over blocks of the reduction axis, with a 128-row operand P
// and a BN-row operand Q in a ring of shared-memory stages and the sums in tensor memory, 32 bits
// each, two accumulators in turn.  The forms differ in what P and Q are and how they lie:
//
//   FORM    P (128 rows)           Q (BN rows)              reduction   D
//   Y       rows of x              rows of w_g              k           rows x n
//   Y_T     rows of w_g            rows of x                k           its transpose: few rows a group
//   DX      rows of dy             columns of w_g           n           rows x k
//   DW      columns of dy_g        columns of x_g           rows of g   n x k of group g
//
// "Rows" lie along the reduction axis (K-major); "columns" lie across it (MN-major): the same
// arrays in place, no transposed copy.  A stage holds 128 bytes of the reduction axis for K-major operands
// (64 values in 16 bits, 128 in 8, 256 in 4), or 64 of its steps as rows of 64 values for
// MN-major ones; both with the 128-byte swizzle of the TMA load.
//
// The work is cut into tiles of D.  Where the groups begin is known on the device only, so every CTA
// (one an SM) adds up the groups' tile counts once and then walks the tiles t = blockIdx.x, +
// gridDim.x, ..., finding each tile's group by bisection.  Warp roles:
//   warp 0      TMA loads of P and Q into the ring (full / empty barriers);
//   warp 1      one thread issues the MMAs; tfull[a] when a tile's are done, tempty[a] before an
//               accumulator's reuse;
//   warps 2, 3  what the loads leave to be done.  Microscaled rows: the scales, in a ring of their own
//               (cfull / cempty), 16 bytes of a row at a time, put into the order that the tensor memory
//               wants (row r of 128 at 16 (r % 32) + 4 (r / 32) of 512 bytes for each 4 blocks).  DW: zeros over the
//               rows past the group's end in its last block, where the load brought the next group's
//               rows (in both operands, since zero times NaN is NaN), reported on fixed[s].
//               Pairs: warp 2 (microscaled rows: warp 13) passes a landed stage on to the leader's fixed[s];
//   warp 12     (microscaled rows) copies landed scales to tensor memory, two chunks in turn (cready / cdone): in
//               the MMA warp the copies and their waits took 300 cycles of the 384 that a stage has;
//   warps 4-11  read D from tensor memory, round once and store.  Rows past the group's end and
//               columns past the width are computed and not stored.
// Pairs (PAIR): two CTAs of a cluster work on one tile of 256 rows of P.  Each loads its own 128 rows
// of P and one half of Q and keeps the sums of its rows; rank 0 issues the MMAs of both, which read
// each half of Q once for the two.  That is what the single form lacks: at 128 x 256 a CTA writes 48 KB into
// shared memory and reads 48 KB out of it for 512 cycles of MMAs, 192 bytes a cycle where an SM has 128;
// in a pair it is 32 + 32 KB (microscaled rows, 128 x 192: 40 + 40 KB for 384 cycles, in a pair 28 + 28).
//
// Measured (device time in a graph, one set of inputs; 65536 x 1152 rows in 32 groups, n = k = 1152, bf16): y 137 us, dx 137,
// dw 142, 1.2 to 1.3 PFLOP/s, the tensor pipe at 75 to 82% of the launch (a plain library product of the same rows and one
// matrix: 159 us); e2m1 8192 x 16384 x 1152 with 16-bit results 97 us, e4m3 144; x 8192 521 and 960 us (4.2 and 2.3
// PFLOP/s). What bounds it: large tiles, shared memory's bandwidth (above); microscaled rows of few stages, the
// results' way out through shared memory; few rows, the reading of w (64 maps of 512 x 1152, 75 MB: 16 us from memory,
// 12 where L2 holds them).
//
// Every wait is bounded: by AG_WAIT_NS where the other side owes a stage or an accumulator, by PR_LONG_NS where it
// may rightly take a whole tile; the latter also ends when a role has given up, in either CTA of a pair
// (pr_fail marks both: what a follower waits for, the leader's MMAs alone commit).  Then the roles run
// out, SMG_PROD_TIMEOUT is set, and the CTA waits (bounded) for its own copies and MMAs before it
// frees the tensor memory.
#pragma once
#include "k_mx.cuh"
#include "tc_util.cuh"
#include "wait_rules.h"

enum { FORM_Y = 0, FORM_YT = 1, FORM_DX = 2, FORM_DW = 3 };

struct ProdArgs {
  const int32_t* off;             // null: one group of all rows
  int n_groups, rows, n, k;
  int p_tiles, q_tiles;           // tiles along the fixed axes (Y, YT, DX: the one in use)
  const uint8_t *sa, *sb;         // scales of microscaled rows, and of the banks
  int pitch;                      // bytes of a row of scales
  uint32_t idesc;
  void* y;
  int64_t ldy, y_stride;
  int y_type;
  bool y_vec;                     // every row of y starts on 16 bytes
  int32_t* err;
};

#define PR_BM 128
#define PR_THREADS(KIND, PAIR) (KIND == 16 ? 384 : PAIR ? 448 : 416)
#define PR_HELPERS 64
#define PR_EPI_WARPS 8
#define PR_SMEM_MAX 232448
#define PR_STAGING (PR_EPI_WARPS * 2048)
#define PR_LONG_NS 60000000000ull   // the longest tile, dw over 2^31 rows, takes 2^25 stages of 512 to 900 cycles: up to 16 s
#define PR_GROUP_BYTES ((3 * SMG_PROD_MAX_GROUPS + 1) * 4)

// KIND 16: f16 or bf16; 8, 4: microscaled
template <int KIND, int BN, bool PAIR>
struct ProdShape {
  static constexpr int QR = PAIR ? BN / 2 : BN;                         // rows of Q that a CTA holds
  static constexpr int QCH = (BN + 127) / 128;                          // 128-row parts of Q
  static constexpr int P_BYTES = PR_BM * 128, Q_BYTES = QR * 128, STAGE = P_BYTES + Q_BYTES;
  // scales come in chunks of 4 words of 4 bytes a row (512 values): 2 (e2m1) or 4 (e4m3) stages
  static constexpr int CHUNK = KIND == 16 ? 0 : (1 + QCH) * 4 * 512, CHUNKS = 3, CHUNK_STAGES = KIND == 4 ? 2 : 4;
  static constexpr int SFC = KIND == 16 ? 0 : (1 + QCH) * 16;           // and their tensor-memory columns, two chunks in turn
  static constexpr int FIXED = CHUNKS * CHUNK + 1024 + PR_STAGING + PR_GROUP_BYTES + 512;
  static constexpr int STAGES = (PR_SMEM_MAX - FIXED) / STAGE > 8 ? 8 : (PR_SMEM_MAX - FIXED) / STAGE;
  static constexpr int SMEM = STAGES * STAGE + FIXED;
  static constexpr int COLS = 2 * BN + 2 * SFC;
  static constexpr int TMEM = 512;   // all of it: its first column is then 0, a constant in every address below
  static_assert(COLS <= 512 && STAGES >= 3, "tile too large");
};

DEV void pr_tma_3d(const CUtensorMap* map, uint64_t* bar, void* dst, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
          ag_smem(dst)),
      "l"((uint64_t)map), "r"(ag_smem(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}

// descriptor of an MN-major operand: 128-byte swizzle, 8-step atoms 1024 bytes apart along the
// reduction axis, blocks of 64 values 8192 bytes apart across it
DEV uint64_t pr_desc_mn(const void* tile) {
  const uint32_t a = ag_smem(tile);
  return (uint64_t)((a >> 4) & 0x3fffu) | (uint64_t)(8192 >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 |
         (uint64_t)2 << 61;
}

// descriptor of 512 bytes of scales for the copy to tensor memory: no swizzle, 8-row parts 128 bytes apart
DEV uint64_t pr_desc_scales(const void* p) {
  const uint32_t a = ag_smem(p);
  return (uint64_t)((a >> 4) & 0x3fffu) | (uint64_t)(128 >> 4) << 16 | (uint64_t)(128 >> 4) << 32 | (uint64_t)1 << 46;
}

template <bool PAIR>
DEV void pr_mma16(uint32_t d, uint64_t p, uint64_t q, uint32_t idesc, uint32_t accum) {
  if constexpr (PAIR)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
        "l"(p), "l"(q), "r"(idesc), "r"(accum));
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
        "l"(p), "l"(q), "r"(idesc), "r"(accum));
}

template <int KIND, bool PAIR>
DEV void pr_mma_mx(uint32_t d, uint64_t p, uint64_t q, uint32_t idesc, uint32_t sp, uint32_t sq, uint32_t accum) {
#define PR_MMA_MX(GROUP, WHAT)                                                                                         \
  asm volatile(                                                                                                        \
      "{\n\t.reg .pred p;\n\t"                                                                                        \
      "setp.ne.b32 p, %6, 0;\n\t"                                                                                     \
      "tcgen05.mma.cta_group::" GROUP ".kind::" WHAT " [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n" ::"r"(d),             \
      "l"(p), "l"(q), "r"(idesc), "r"(sp), "r"(sq), "r"(accum))
  if constexpr (KIND == 4 && PAIR) PR_MMA_MX("2", "mxf4.block_scale.scale_vec::2X");
  else if constexpr (KIND == 4) PR_MMA_MX("1", "mxf4.block_scale.scale_vec::2X");
  else if constexpr (PAIR) PR_MMA_MX("2", "mxf8f6f4.block_scale.scale_vec::1X");
  else PR_MMA_MX("1", "mxf8f6f4.block_scale.scale_vec::1X");
#undef PR_MMA_MX
}

// 512 bytes of scales to tensor memory (PAIR: of each CTA to its own)
template <bool PAIR>
DEV void pr_copy_scales(uint32_t tmem, const void* p) {
  if constexpr (PAIR)
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(pr_desc_scales(p)) : "memory");
  else
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(pr_desc_scales(p)) : "memory");
}

// true in one lane of a converged warp
DEV bool pr_elect() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}

DEV void pr_proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
DEV void pr_arrive(uint64_t* b) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(ag_smem(b)) : "memory"); }

// ---- the pair of CTAs (a cluster of 2): rank 0 issues the MMAs of both ----
DEV uint32_t pr_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}

// Arrival on the leader's barrier that lies where b does here, and what the leader does once it has seen it (ag_wait<true>
// or pr_test<true>): release and acquire at cluster scope, since what it reports is this CTA's shared memory (landed
// copies, scales, the zeros of dw's last block) for instructions that the leader issues.  The fences are
// restricted to shared memory (arrivals with CTA scope, which PTX does not promise to be enough, took 1 to 4% less:
// 8192 x 16384 x 1152 in 4 bits 95 us against 97, in 8 bits 139 against 144); full ones also wait for the results that
// the CTA is storing (on every stage the products ran at 0.4 of their speed, on the scales alone 131 us).
DEV void pr_arrive_leader(uint64_t* b) {
  asm volatile(
      "{\n\t.reg .b32 a;\n\t"
      "fence.release.sync_restrict::shared::cta.cluster;\n\t"
      "mapa.shared::cluster.u32 a, %0, 0;\n\t"
      "mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [a];\n\t}\n" ::"r"(ag_smem(b))
      : "memory");
}
DEV void pr_acquire_pair() { asm volatile("fence.acquire.sync_restrict::shared::cluster.cluster;" ::: "memory"); }

// arrives on b here (PAIR: there and here) when the MMAs issued so far are done
template <bool PAIR>
DEV void pr_commit(uint64_t* b) {
  if constexpr (PAIR)
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(ag_smem(b)),
                 "h"((uint16_t)3)
                 : "memory");
  else
    ag_commit(b);
}

template <bool PAIR>
DEV void pr_cluster_sync() {
  if constexpr (PAIR)
    asm volatile(
        "barrier.cluster.arrive.release.aligned;\n\t"
        "barrier.cluster.wait.acquire.aligned;" ::
            : "memory");
}

// whether the phase is over, without waiting
template <bool CLUSTER>
DEV bool pr_test(uint64_t* b, uint32_t parity) {
  uint32_t ok;
  if constexpr (CLUSTER)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.relaxed.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}\n"
        : "=r"(ok)
        : "r"(ag_smem(b)), "r"(parity)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}\n"
        : "=r"(ok)
        : "r"(ag_smem(b)), "r"(parity)
        : "memory");
  return ok != 0;
}

// A role gives up: every role of this CTA, and of the other one of a pair, is told.  (The other CTA is there: both
// meet at a cluster barrier before the first and after the last role.)
template <bool PAIR>
DEV void pr_fail(volatile int* failed) {
  *failed = 1;
  if constexpr (PAIR)
    asm volatile(
        "{\n\t.reg .b32 a;\n\t"
        "mapa.shared::cluster.u32 a, %0, %1;\n\t"
        "st.relaxed.cluster.shared::cluster.u32 [a], %2;\n\t}\n" ::"r"(ag_smem((const void*)failed)),
        "r"(pr_rank() ^ 1u), "r"(1)
        : "memory");
}

DEV bool pr_wait_long(uint64_t* b, uint32_t parity, volatile int* failed) {
  return wait_long([&] { return ag_wait(b, parity); }, [&] { return *failed != 0; }, ag_now, PR_LONG_NS);
}

// what every role knows of the tiles
struct ProdTiles {
  const int *beg, *end, *cum;   // first row, row past the last, and first row tile of each group
  int n_groups, fixed;          // tiles of a row tile along the fixed axes
  int total, first, step;       // this CTA's (pair's) place among the `step` that walk the tiles
  // The r-th tile of this CTA (>= total: none).  DW's tiles are as long as their groups, the longest first
  // and every other round of them backwards, so that no CTA has the longest of every round.
  template <int FORM>
  DEV int at(int r) const {
    return r * step + (FORM == FORM_DW && (r & 1) ? step - 1 - first : first);
  }
};

struct ProdTile {
  int g, r0, r1;                // group, first row of the tile, row past the group's last
  int f;                        // index along the fixed axes
  DEV ProdTile uniform() const {
    ProdTile t;
    t.g = __shfl_sync(0xffffffffu, g, 0);
    t.r0 = __shfl_sync(0xffffffffu, r0, 0);
    t.r1 = __shfl_sync(0xffffffffu, r1, 0);
    t.f = __shfl_sync(0xffffffffu, f, 0);
    return t;
  }
};

template <int FORM, int BN, bool PAIR>
DEV ProdTile prod_tile(const ProdTiles& T, int t) {
  const int u = t / T.fixed;
  ProdTile r;
  r.f = t - u * T.fixed;
  if (FORM == FORM_DW) {        // T.cum: the groups in order of length
    r.g = T.cum[u];
    r.r0 = T.beg[r.g];
    r.r1 = T.end[r.g];
    return r;
  }
  int lo = 0, hi = T.n_groups;  // the last group whose first row tile is <= u (empty groups have none)
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (T.cum[mid] <= u) lo = mid;
    else hi = mid;
  }
  r.g = lo;
  r.r0 = T.beg[lo] + (u - T.cum[lo]) * (FORM == FORM_YT ? BN : PAIR ? 2 * PR_BM : PR_BM);
  r.r1 = T.end[lo];
  return r;
}

template <int KIND, int BN, int FORM, bool PAIR>
__global__ void __launch_bounds__(PR_THREADS(KIND, PAIR), 1)
    k_prod(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const __grid_constant__ ProdArgs g) {
  using S = ProdShape<KIND, BN, PAIR>;
  static_assert(!PAIR || FORM != FORM_YT, "pairs: rows as P");
  constexpr int STAGES = S::STAGES;
  constexpr bool P_MN = FORM == FORM_DW, Q_MN = FORM == FORM_DX || FORM == FORM_DW;
  constexpr int BK = P_MN || Q_MN ? 64 : 1024 / KIND;   // values of the reduction axis in a stage
  constexpr int SUB = BK / 4;                           // and in an MMA
  constexpr bool RELAY = PAIR || FORM == FORM_DW;       // every landed stage is passed on
  constexpr int RELAYS = FORM == FORM_DW ? PR_HELPERS / 32 : 1, RELAY_WARP = KIND == 16 ? 2 : 13;   // by so many warps from this one
  extern __shared__ unsigned char pr_raw[];
  unsigned char* base = (unsigned char*)(((uintptr_t)pr_raw + 1023) & ~(uintptr_t)1023);
  unsigned char* sP = base;
  unsigned char* sQ = sP + STAGES * S::P_BYTES;
  unsigned char* sS = sQ + STAGES * S::Q_BYTES;
  unsigned char* staging = sS + S::CHUNKS * S::CHUNK;
  int* s_beg = (int*)(staging + PR_STAGING);
  int* s_end = s_beg + SMG_PROD_MAX_GROUPS;
  int* s_cum = s_end + SMG_PROD_MAX_GROUPS;
  uint64_t* full = (uint64_t*)(((uintptr_t)(s_cum + SMG_PROD_MAX_GROUPS + 1) + 7) & ~(uintptr_t)7);
  uint64_t* empty = full + STAGES;
  uint64_t* fixed = empty + STAGES;
  uint64_t* cfull = fixed + STAGES;      // microscaled rows: a chunk of scales has landed,
  uint64_t* cempty = cfull + S::CHUNKS;  // has been copied to tensor memory,
  uint64_t* cdone = cempty + S::CHUNKS;  // and the MMAs that use the copy are done
  uint64_t* cready = cdone + 2;          // the copy is in tensor memory
  uint64_t* cpeer = cready + 2;          // PAIR: the other CTA's chunk has landed
  uint64_t* tfull = cpeer + S::CHUNKS;
  uint64_t* tempty = tfull + 2;
  uint64_t* done = tempty + 2;
  uint32_t* tmem_slot = (uint32_t*)(done + 1);
  __shared__ int sh_fail;
  volatile int* failed = &sh_fail;
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;

  if (tid == 32) {   // the tensor maps are on their way while the rest is set up
    asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)&tmA) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)&tmB) : "memory");
  }
  if (tid == 0) {
    for (int s = 0; s < STAGES; ++s) {
      ag_mbar_init(&full[s], 1);
      ag_mbar_init(&empty[s], 1);
      ag_mbar_init(&fixed[s], RELAYS * (PAIR ? 2 : 1));
    }
    for (int s = 0; s < S::CHUNKS; ++s) {
      ag_mbar_init(&cfull[s], PR_HELPERS);
      ag_mbar_init(&cempty[s], 1);
      ag_mbar_init(&cpeer[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      ag_mbar_init(&cdone[a], 1);
      ag_mbar_init(&cready[a], 1);
      ag_mbar_init(&tfull[a], 1);
      ag_mbar_init(&tempty[a], PR_EPI_WARPS * (PAIR ? 2 : 1));
    }
    ag_mbar_init(done, KIND == 16 ? 1 : 2);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    sh_fail = 0;
  }
  __syncwarp();
  pr_cluster_sync<PAIR>();   // the other's barriers exist
  if (warp == 2) {
    if constexpr (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(ag_smem(tmem_slot)), "r"(S::TMEM)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(ag_smem(tmem_slot)), "r"(S::TMEM)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  }
  heads_next();
  heads_wait();   // barriers and tensor memory are set up; from here on global memory is read
  // groups: offsets that break the rules are reported, and every group is then taken as empty
  int bad = 0;
  for (int i = tid; i < g.n_groups; i += PR_THREADS(KIND, PAIR)) {
    int a = 0, b = g.rows;
    if (g.off) {
      a = g.off[i];
      b = g.off[i + 1];
      bad |= a < 0 || b < a || b > g.rows || (i == 0 && a != 0) || (i == g.n_groups - 1 && b != g.rows);
    }
    s_beg[i] = a;
    s_end[i] = b;
  }
  ag_fence_before();
  bad = __syncthreads_or(bad);
  ag_fence_after();
  if (bad) {
    if (tid == 0 && blockIdx.x == 0 && g.err) atomicOr(g.err, SMG_PROD_OFFSETS);
    for (int i = tid; i < g.n_groups; i += PR_THREADS(KIND, PAIR)) s_beg[i] = s_end[i] = 0;
    __syncthreads();
  }
  constexpr uint32_t tmem = 0;
  if (tid == 0 && *tmem_slot != tmem) pr_fail<PAIR>(failed);
  constexpr int RT = FORM == FORM_YT ? BN : PAIR ? 2 * PR_BM : PR_BM;
  const int rank = PAIR ? (int)pr_rank() : 0;   // which of a pair's 128 rows of P (and halves of Q) are this CTA's
  if (FORM == FORM_DW) {   // groups by length (beyond 256 of them, where no single one holds the end up, as they come)
    for (int i = tid; i < g.n_groups; i += PR_THREADS(KIND, PAIR)) {
      int place = i;
      if (g.n_groups <= 256) {
        const int len = s_end[i] - s_beg[i];
        place = 0;
        for (int o = 0; o < g.n_groups; ++o) {
          const int other = s_end[o] - s_beg[o];
          place += other > len || (other == len && o < i);
        }
      }
      s_cum[place] = i;
    }
  } else if (warp == 0) {   // first row tile of every group
    int at = 0;
    for (int i0 = 0; i0 < g.n_groups; i0 += 32) {
      const int i = i0 + lane;
      const int own = i >= g.n_groups ? 0 : (s_end[i] - s_beg[i] + RT - 1) / RT;
      int sum = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += v;
      }
      if (i < g.n_groups) s_cum[i] = at + sum - own;
      at += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (lane == 0) s_cum[g.n_groups] = at;
  }
  __syncthreads();
  ProdTiles T;
  T.beg = s_beg; T.end = s_end; T.cum = s_cum;
  T.n_groups = g.n_groups;
  T.fixed = FORM == FORM_DW ? g.p_tiles * g.q_tiles : FORM == FORM_YT ? g.p_tiles : g.q_tiles;
  T.total = __shfl_sync(0xffffffffu, *failed ? 0 : (FORM == FORM_DW ? g.n_groups : s_cum[g.n_groups]) * T.fixed, 0);
  T.first = PAIR ? blockIdx.x >> 1 : blockIdx.x;
  T.step = PAIR ? gridDim.x >> 1 : gridDim.x;
  const int red = FORM == FORM_DX ? g.n : g.k;   // (DW: the group's rows)
  bool ok = true;

  // The loads and the MMAs are issued by one elected lane, in code that the whole warp runs and whose branches
  // the compiler can see to be the warp's (votes, values handed on by a shuffle): their operands live in
  // uniform registers.  From a single thread's own code each MMA took 115 cycles to issue whatever its
  // width, a block-scaled one with branches on values out of shared memory 220 (32 to 128 are needed).
  // A pair's last tile with no more than half of its columns: MMAs of half the width
  const auto slim = [&](const ProdTile& c) {
    return PAIR && (FORM == FORM_Y ? g.n : g.k) - (FORM == FORM_DW ? c.f / g.p_tiles : c.f) * BN <= BN / 2;
  };
  const auto wait = [](uint64_t* b, uint32_t parity) { return __all_sync(0xffffffffu, ag_wait(b, parity)) != 0; };
  // for arrivals from either CTA of a pair
  const auto wait_pair = [](uint64_t* b, uint32_t parity) {
    const bool over = __all_sync(0xffffffffu, ag_wait<PAIR>(b, parity)) != 0;
    if (PAIR) pr_acquire_pair();
    return over;
  };
  if (warp == 0) {   // loads
    const bool one = pr_elect();
    uint32_t it = 0;
    for (int r = 0, t; (t = T.template at<FORM>(r)) < T.total && ok; ++r) {
      const ProdTile c = prod_tile<FORM, BN, PAIR>(T, t).uniform();
      const int nk = ((FORM == FORM_DW ? c.r1 - c.r0 : red) + BK - 1) / BK;
      const int half = rank * (slim(c) ? S::QR / 2 : S::QR);   // where this CTA's part of Q begins
      for (int kb = 0; kb < nk; ++kb, ++it) {
        const int s = (int)(it % STAGES);
        if (it >= STAGES && !wait(&empty[s], ((it / STAGES) & 1u) ^ 1u)) { ok = false; break; }
        unsigned char *p = sP + s * S::P_BYTES, *q = sQ + s * S::Q_BYTES;
        if (!one) continue;
        ag_expect_tx(&full[s], S::STAGE);
        const int x = KIND == 16 ? kb * BK : kb * 128;   // microscaled rows are loaded as bytes
        if (FORM == FORM_Y) {
          ag_tma_2d(&tmA, &full[s], p, x, c.r0 + rank * PR_BM);
          pr_tma_3d(&tmB, &full[s], q, x, c.f * BN + half, c.g);
        } else if (FORM == FORM_YT) {
          pr_tma_3d(&tmB, &full[s], p, x, c.f * PR_BM, c.g);
          ag_tma_2d(&tmA, &full[s], q, x, c.r0);
        } else if (FORM == FORM_DX) {
          ag_tma_2d(&tmA, &full[s], p, x, c.r0 + rank * PR_BM);
#pragma unroll
          for (int j = 0; j < S::QR / 64; ++j) pr_tma_3d(&tmB, &full[s], q + j * 8192, c.f * BN + half + j * 64, x, c.g);
        } else {
          const int m0 = c.f % g.p_tiles * RT + rank * PR_BM, n0 = c.f / g.p_tiles * BN + half;
#pragma unroll
          for (int j = 0; j < PR_BM / 64; ++j) ag_tma_2d(&tmA, &full[s], p + j * 8192, m0 + j * 64, c.r0 + x);
#pragma unroll
          for (int j = 0; j < S::QR / 64; ++j) ag_tma_2d(&tmB, &full[s], q + j * 8192, n0 + j * 64, c.r0 + x);
        }
      }
    }
    // the last loads must have landed before the CTA ends
    for (uint32_t j = it > STAGES ? it - STAGES : 0; j < it; ++j) ok = wait(&full[j % STAGES], (j / STAGES) & 1u) && ok;
    if (!ok) pr_fail<PAIR>(failed);
  } else if (warp == 1 && rank == 0) {   // MMAs
    const bool one = pr_elect();
    uint32_t it = 0, j = 0, ci = 0;
    bool ready = false;
    for (int t; (t = T.template at<FORM>(j)) < T.total && ok; ++j) {
      const ProdTile c = prod_tile<FORM, BN, PAIR>(T, t).uniform();
      const int len = FORM == FORM_DW ? c.r1 - c.r0 : red, nk = (len + BK - 1) / BK;
      const uint32_t acc = j & 1u;
      if (j >= 2 && !wait_pair(&tempty[acc], ((j >> 1) & 1u) ^ 1u)) { ok = false; break; }
      ag_fence_after();
      const uint32_t d = tmem + acc * BN;
      const uint32_t idesc = slim(c) ? (g.idesc & ~(0x3fu << 17)) | (uint32_t)(BN / 16) << 17 : g.idesc;
      for (int kb = 0; kb < nk; ++kb, ++it) {
        const int s = (int)(it % STAGES);
        const uint32_t ph = (it / STAGES) & 1u;
        const int left = len - kb * BK;
        uint64_t* landed = RELAY ? fixed : full;
        if (!__all_sync(0xffffffffu, ready)) {
          if (!(RELAY ? wait_pair(&landed[s], ph) : wait(&landed[s], ph))) { ok = false; break; }
        } else if (PAIR) {
          pr_acquire_pair();   // the arrivals that pr_test saw
        }
        if (KIND != 16 && kb % S::CHUNK_STAGES == 0 && !wait(&cready[ci & 1u], (ci >> 1) & 1u)) { ok = false; break; }
        ready = pr_test<PAIR>(&landed[(it + 1) % STAGES], ((it + 1) / STAGES) & 1u);   // the next stage, while this one's MMAs go out
        ag_fence_after();
        const unsigned char *p = sP + s * S::P_BYTES, *q = sQ + s * S::Q_BYTES;
        const uint64_t dp = P_MN ? pr_desc_mn(p) : ag_desc(p), dq = Q_MN ? pr_desc_mn(q) : ag_desc(q);
        const int subs = left >= BK ? 4 : (left + SUB - 1) / SUB;
        if (one) {
          if constexpr (KIND == 16) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (i < subs) pr_mma16<PAIR>(d, dp + i * (P_MN ? 128 : 2), dq + i * (Q_MN ? 128 : 2), idesc, (kb | i) != 0);
          } else {
            const uint32_t tp = tmem + 2 * BN + (ci & 1u) * S::SFC, tq = tp + 16;
            const uint32_t w0 = KIND == 4 ? kb % 2 * 2 : kb % 4;   // the stage's first word of the chunk
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if (i < subs) {
                // an MMA's 2 scales of a row (e2m1) are half a word, its one (e4m3) is a byte of it
                const uint32_t w = w0 + (KIND == 4 ? i / 2 : 0), id = KIND == 4 ? (i & 1) * 2 : i;
                pr_mma_mx<KIND, PAIR>(d, dp + i * 2, dq + i * 2, idesc | id << 29 | id << 4, tp + 4 * w, tq + 4 * S::QCH * w, (kb | i) != 0);
              }
            }
            if (kb % S::CHUNK_STAGES == S::CHUNK_STAGES - 1 || kb == nk - 1) pr_commit<PAIR>(&cdone[ci & 1u]);
          }
          pr_commit<PAIR>(&empty[s]);
        }
        if (KIND != 16 && (kb % S::CHUNK_STAGES == S::CHUNK_STAGES - 1 || kb == nk - 1)) ++ci;
      }
      if (one) pr_commit<PAIR>(&tfull[acc]);   // after a failed wait too: arrives when the issued MMAs are done
    }
    if (one) pr_commit<PAIR>(done);   // every issued MMA has completed before the tensor memory is freed
    if (!wait(done, 0) || !ok) pr_fail<PAIR>(failed);
  } else if (warp == 12) {   // microscaled rows: scales from shared to tensor memory
    const bool one = pr_elect();
    uint32_t ci = 0;
    const int chunks = (red + 511) / 512;
    for (int r = 0, t; (t = T.template at<FORM>(r)) < T.total && ok; ++r) {
      for (int i = 0; i < chunks; ++i, ++ci) {
        const uint32_t s = ci % S::CHUNKS, ph = (ci / S::CHUNKS) & 1u;
        if (rank == 0 && ci >= 2 && !wait(&cdone[ci & 1u], ((ci >> 1) & 1u) ^ 1u)) { ok = false; break; }
        if (!wait(&cfull[s], ph)) { ok = false; break; }
        pr_proxy_fence();   // they were written by ordinary copies
        if (PAIR && rank == 1) {
          if (one) pr_arrive_leader(&cpeer[s]);
          continue;
        }
        if (PAIR && !wait_pair(&cpeer[s], ph)) { ok = false; break; }
        ag_fence_after();
        if (one) {
          const unsigned char* sc = sS + s * S::CHUNK;
          const uint32_t tp = tmem + 2 * BN + (ci & 1u) * S::SFC;
#pragma unroll
          for (int k = 0; k < 4 * (1 + S::QCH); ++k) pr_copy_scales<PAIR>(tp + 4 * k, sc + 512 * k);
          pr_commit<PAIR>(&cempty[s]);
          pr_commit<PAIR>(&cready[ci & 1u]);
        }
      }
    }
    if (one && rank == 0) pr_commit<PAIR>(done);
    if (!ok) pr_fail<PAIR>(failed);
  } else if (KIND != 16 && (warp == 2 || warp == 3)) {   // scales to shared memory
    const int h = tid - 64;
    uint32_t it = 0;
    for (int r = 0, t; (t = T.template at<FORM>(r)) < T.total && ok; ++r) {
      const ProdTile c = prod_tile<FORM, BN, PAIR>(T, t);
      // rows of w_g and rows of x, whichever is P
      const int w0 = c.f * (FORM == FORM_YT ? PR_BM : BN);
      const int p_lim = FORM == FORM_YT ? g.n - w0 : c.r1 - c.r0 - rank * PR_BM, q_lim = FORM == FORM_YT ? c.r1 - c.r0 : g.n - w0;
      const int64_t wr = (int64_t)c.g * g.n + w0, xr = c.r0 + rank * PR_BM;
      const uint8_t* ps = (FORM == FORM_YT ? g.sb + wr * g.pitch : g.sa + xr * g.pitch);
      const uint8_t* qs = (FORM == FORM_YT ? g.sa + xr * g.pitch : g.sb + wr * g.pitch);
      // 8 rows x 16 bytes a warp and step: thread h has word h % 4 of the rows h / 4, h / 4 + 16, ...
      const int r0 = h >> 2, w = h & 3;
      for (int k0 = 0; k0 < g.pitch; k0 += 16, ++it) {
        const uint32_t s = it % S::CHUNKS;
        if (it >= S::CHUNKS && !ag_wait(&cempty[s], ((it / S::CHUNKS) & 1u) ^ 1u)) { ok = false; break; }
        const uint32_t sc = ag_smem(sS + s * S::CHUNK);
        if (k0 + 4 * w < g.pitch) {
#pragma unroll
          for (int i = 0; i < (PR_BM + BN) / 16; ++i) {
            const bool is_p = i < PR_BM / 16;
            const int r = r0 + 16 * (is_p ? i : i - PR_BM / 16);
            const uint32_t part = is_p ? w : 4 + w * S::QCH + (r >> 7);
            // (the scales of rows that are not there are left as they are: they touch only what is not stored)
            if (r < (is_p ? p_lim : q_lim))
              asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(sc + 512 * part + (r & 31) * 16 + ((r >> 5) & 3) * 4),
                           "l"((is_p ? ps : qs) + (int64_t)r * g.pitch + k0 + 4 * w)
                           : "memory");
          }
        }
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(ag_smem(&cfull[s])) : "memory");
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (!ok) pr_fail<PAIR>(failed);
  } else if (RELAY && warp >= RELAY_WARP && warp < RELAY_WARP + RELAYS) {   // landed stages, passed on
    const int h = tid - RELAY_WARP * 32;
    uint32_t it = 0;
    for (int r = 0, t; (t = T.template at<FORM>(r)) < T.total && ok; ++r) {
      const ProdTile c = prod_tile<FORM, BN, PAIR>(T, t);
      const int len = FORM == FORM_DW ? c.r1 - c.r0 : red;
      // every block is passed on, whole or not: a wait that skipped blocks could not tell a
      // stage's next filling from the one after
      for (int k0 = 0; k0 < len; k0 += BK, ++it) {
        const int s = (int)(it % STAGES), tail = len - k0;
        if (!__all_sync(0xffffffffu, pr_wait_long(&full[s], (it / STAGES) & 1u, failed))) { ok = false; break; }
        if (FORM == FORM_DW && tail < BK) {
          // steps tail .. of every block of 64 values, up to the last that an MMA reads: 128 bytes each, the
          // swizzle stays within them
          const int v = (h & 7) * 16, last = (tail + SUB - 1) / SUB * SUB;
          for (int k = tail + (h >> 3); k < last; k += PR_HELPERS / 8) {
#pragma unroll
            for (int b = 0; b < PR_BM / 64; ++b) *(uint4*)(sP + s * S::P_BYTES + b * 8192 + k * 128 + v) = make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int b = 0; b < S::QR / 64; ++b) *(uint4*)(sQ + s * S::Q_BYTES + b * 8192 + k * 128 + v) = make_uint4(0, 0, 0, 0);
          }
          pr_proxy_fence();
        }
        __syncwarp();
        if (lane == 0) {
          if (PAIR) pr_arrive_leader(&fixed[s]);
          else pr_arrive(&fixed[s]);
        }
      }
    }
    if (!ok) pr_fail<PAIR>(failed);
  } else if (warp >= 4 && warp < 12) {   // results
    const int ew = warp - 4, quarter = ew & 3, half = ew >> 2;
    unsigned char* stg = staging + ew * 2048;
    uint32_t j = 0;
    for (int t; (t = T.template at<FORM>(j)) < T.total; ++j) {
      const ProdTile c = prod_tile<FORM, BN, PAIR>(T, t);
      const uint32_t acc = j & 1u;
      if (!__all_sync(0xffffffffu, pr_wait_long(&tfull[acc], (j >> 1) & 1u, failed) && !*failed)) {
        if (lane == 0) pr_fail<PAIR>(failed);
        break;
      }
      ag_fence_after();
      const bool none = FORM == FORM_DW && c.r1 == c.r0;   // an empty group: zeros
      const uint32_t d = tmem + acc * BN + ((uint32_t)(quarter * 32) << 16);
      // tile's place in y: rows row0 .. row_lim - 1, columns col0 .. col_lim - 1
      const int row0 = (FORM == FORM_DW ? c.f % g.p_tiles * RT : c.r0) + rank * PR_BM, row_lim = FORM == FORM_DW ? g.n : c.r1;
      const int col0 = FORM == FORM_DW ? c.f / g.p_tiles * BN : c.f * (FORM == FORM_YT ? PR_BM : BN);
      const int col_lim = FORM == FORM_Y || FORM == FORM_YT ? g.n : g.k;
      const int64_t y0 = FORM == FORM_DW ? (int64_t)c.g * g.y_stride : 0;
      if (FORM != FORM_YT && BN >= 64 && g.y_type != SMG_EMB_F32 && g.y_vec && col0 + BN <= col_lim && !none) {
        // 16-bit results of a tile that is whole in its columns: the places of the lane's 4 rows are found once
        const int q = lane & 3, r0 = lane >> 2;
        uint16_t* o = (uint16_t*)g.y + y0 + (int64_t)(row0 + quarter * 32 + r0) * g.ldy + col0 + half * (BN / 2) + q * 8;
        const int64_t step = 8 * g.ldy;
        const int left = row_lim - row0 - quarter * 32 - r0;   // rows r0 + 8 i below it are there
        unsigned char* in = stg + r0 * 64 + ((q ^ (r0 >> 1)) & 3) * 16;
        const bool bf = g.y_type == SMG_EMB_BF16;
#pragma unroll 1
        for (int c = 0; c < BN / 2; c += 32) {
          uint32_t v[32], w[16];
          ag_tmem_ld32(d + half * (BN / 2) + c, v);
          if (bf) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const __nv_bfloat162 b = __floats2bfloat162_rn(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
              w[i] = *(const uint32_t*)&b;
            }
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const __half2 b = __floats2half2_rn(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
              w[i] = *(const uint32_t*)&b;
            }
          }
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 4; ++i)
            *(uint4*)(stg + lane * 64 + ((i ^ (lane >> 1)) & 3) * 16) = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 4; ++i)   // 8 rows on, the swap of parts is the same: (r + 8) / 2 = r / 2 + 4
            if (8 * i < left) *(uint4*)(o + i * step + c) = *(const uint4*)(in + i * 512);
        }
        ag_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (PAIR) pr_arrive_leader(&tempty[acc]);
          else pr_arrive(&tempty[acc]);
        }
        continue;
      }
      constexpr int HALF = BN >= 64 ? BN / 2 : BN;         // columns of D that a warp takes
      if (BN >= 64 || half == 0) {
        for (int c0 = half * HALF; c0 < half * HALF + HALF; c0 += 32) {
          if (FORM == FORM_YT) {
            if (row0 + c0 >= row_lim) break;
          } else if (col0 + c0 >= col_lim) {
            break;
          }
          uint32_t v[32];
          if (none) {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = 0;
          } else {
            ag_tmem_ld32(d + c0, v);
          }
          if (FORM == FORM_YT) {   // lane: a column of y; v[i]: row row0 + c0 + i
            const int colb = col0 + quarter * 32;
            if (g.y_type == SMG_EMB_F32 || !g.y_vec || colb + 32 > col_lim) {   // 32 neighbouring values of a row a step
              const int col = colb + lane;
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                const int row = row0 + c0 + i;
                if (row < row_lim && col < col_lim) {
                  const int64_t at = (int64_t)row * g.ldy + col;
                  const float f = __uint_as_float(v[i]);
                  if (g.y_type == SMG_EMB_F32) ((float*)g.y)[at] = f;
                  else if (g.y_type == SMG_EMB_BF16) ((__nv_bfloat16*)g.y)[at] = __float2bfloat16_rn(f);
                  else ((__half*)g.y)[at] = __float2half_rn(f);
                }
              }
            } else {   // through shared memory, 32 rows of 64 bytes: 8 rows x 64 bytes a step
              __syncwarp();
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                const float f = __uint_as_float(v[i]);
                uint16_t u;
                if (g.y_type == SMG_EMB_BF16) u = __bfloat16_as_ushort(__float2bfloat16_rn(f));
                else u = __half_as_ushort(__float2half_rn(f));
                ((uint16_t*)stg)[i * 32 + lane] = u;
              }
              __syncwarp();
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int r = i * 8 + (lane >> 2), row = row0 + c0 + r;
                if (row < row_lim)
                  *(uint4*)((uint16_t*)g.y + (int64_t)row * g.ldy + colb + (lane & 3) * 8) = *(const uint4*)(stg + r * 64 + (lane & 3) * 16);
              }
            }
          } else {
            // through shared memory: rows of 64 bytes (32 values of 16 bits, or 16 of 32), 16-byte parts swapped about by the
            // row, so that both a lane's own row and 8 rows side by side meet no bank twice
            const int per = g.y_type == SMG_EMB_F32 ? 16 : 32;
            for (int h0 = 0; h0 < 32; h0 += per) {
              uint32_t w[16];
              if (g.y_type == SMG_EMB_F32) {
#pragma unroll
                for (int i = 0; i < 16; ++i) w[i] = h0 ? v[16 + i] : v[i];
              } else if (g.y_type == SMG_EMB_BF16) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                  const __nv_bfloat162 b = __floats2bfloat162_rn(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
                  w[i] = *(const uint32_t*)&b;
                }
              } else {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                  const __half2 b = __floats2half2_rn(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
                  w[i] = *(const uint32_t*)&b;
                }
              }
              __syncwarp();
#pragma unroll
              for (int q = 0; q < 4; ++q)
                *(uint4*)(stg + lane * 64 + ((q ^ (lane >> 1)) & 3) * 16) = make_uint4(w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]);
              __syncwarp();
              const int size = g.y_type == SMG_EMB_F32 ? 4 : 2, each = 16 / size;
              if (!g.y_vec) {
                // rows of y off 16 bytes: 32 (16 bits) or 2 x 16 neighbouring values a step, so that a store still fills
                // whole sectors (value by value in the 16-byte order below it touched five times as many)
                const int left = row_lim - row0 - quarter * 32, top = col0 + c0 + h0;   // rows and columns from here
                const int64_t at = y0 + (int64_t)(row0 + quarter * 32) * g.ldy + top;
                if (size == 2) {
                  uint16_t* o = (uint16_t*)g.y + at + lane;
                  const unsigned char* in = stg + (lane & 7) * 2;
                  if (top + lane < col_lim) {
#pragma unroll
                    for (int r = 0; r < 32; ++r, o += g.ldy)
                      if (r < left) *o = *(const uint16_t*)(in + r * 64 + (((lane >> 3) ^ (r >> 1)) & 3) * 16);
                  }
                } else {
                  const int e = lane & 15, r0 = lane >> 4;
                  uint32_t* o = (uint32_t*)g.y + at + r0 * g.ldy + e;
                  const unsigned char* in = stg + r0 * 64 + (e & 3) * 4;
                  if (top + e < col_lim) {
#pragma unroll
                    for (int r = 0; r < 32; r += 2, o += 2 * g.ldy)
                      if (r + r0 < left) *o = *(const uint32_t*)(in + r * 64 + (((e >> 2) ^ (r >> 1)) & 3) * 16);
                  }
                }
                continue;
              }
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int r = i * 8 + (lane >> 2), q = lane & 3;
                const int row = row0 + quarter * 32 + r, col = col0 + c0 + h0 + q * each;
                if (row >= row_lim || col >= col_lim) continue;
                const uint4 u = *(const uint4*)(stg + r * 64 + ((q ^ (r >> 1)) & 3) * 16);
                unsigned char* o = (unsigned char*)g.y + (y0 + (int64_t)row * g.ldy + col) * size;
                if (col + each <= col_lim) {
                  *(uint4*)o = u;
                } else {
                  const uint32_t uw[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                  for (int e = 0; e < 8; ++e) {
                    if (e >= each || col + e >= col_lim) break;
                    if (size == 4) ((uint32_t*)o)[e] = uw[e & 3];
                    else ((uint16_t*)o)[e] = (uint16_t)(uw[e >> 1] >> (16 * (e & 1)));
                  }
                }
              }
            }
          }
        }
      }
      ag_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (PAIR) pr_arrive_leader(&tempty[acc]);
        else pr_arrive(&tempty[acc]);
      }
    }
  }
  __syncwarp();
  ag_fence_before();
  __syncthreads();
  pr_cluster_sync<PAIR>();   // neither CTA leaves while the other's MMAs or arrivals may still reach it
  if (tid == 0 && *failed && g.err) atomicOr(g.err, SMG_PROD_TIMEOUT);
  if (warp == 2) {
    ag_fence_after();
    if constexpr (PAIR)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::TMEM) : "memory");
    else
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::TMEM) : "memory");
  }
}
