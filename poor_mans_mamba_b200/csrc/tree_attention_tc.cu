// Attention of drafted tokens over a paged cache on the fifth-generation tensor cores (the formulas of tree_attention.cu;
// bfloat16, head size 64 or 128, pages of a multiple of 8 positions).
//
// A unit of work is up to 128 rows, or 256 (a row: a token and a query head of the group), of ONE request and ONE key/value
// head; its keys are tiles of 128, first the request's cached keys, then its own tokens of this step.  The number of tiles of
// all units is only known on the device (lengths are tensors, contexts are ragged), so every block adds it up and takes an
// equal share of the tiles, one behind the other (148 SMs stay busy to the end whatever the batch).  A unit that lies within one
// share is finished by its block; of a unit that shares cut, every block leaves (maximum, sum, unnormalised result) in scratch
// and a second launch merges them in the order of the keys, so results do not depend on which block came first.
// Within a block warp 0 brings K and V tiles by TMA (cached keys in boxes that lie inside a page, the step's own from k and
// v) into a ring; two sets of four warps turn S = Q K^T into P, a thread a row, 64 of its scores at a time in registers, so that
// maximum and sum need no other thread; and for each set a warp issues S and O += P V.  Units of 128 rows: the sets take the
// tiles in turn, and their results are joined when the unit ends.  Units of 256: every set has 128 rows, and K and V are brought
// once for both (16 requests of 8,192 with trees of 64, 64 / 8 heads of 128: 308 us, in units of 128 331; 144 rows a unit: 32 and 33).
// Each set has its S, running maximum and sum, and its O in tensor memory (4 x 128 columns); P takes the place of the S that it is
// made from.  S and P go in halves of 64 keys, each with barriers of its own: while one half's exponentials are made, the other
// half's P V and the S behind it run, so neither side waits for the other's answer (whole tiles: 385 us where halves take 305).
// The ring and the products run on across units.
// What bounds half a tile of two sets, 256 rows and 64 keys, clocks: products 1,259 (the S of 64 columns read Q at 128 bytes a clock:
// 48 each instead of 32), exponentials 1,024 (16 a clock), 32 KB from L2 at 5.4 TB/s of all blocks 1,450; it takes 2,250, of them 2,000 a
// warp's own way through load, maximum, exponentials and store: two warps a scheduler do not cover each other's latencies.  With
// units of 128 rows memory bounds it: 32 x 16,384 takes 245 us, the copies alone 237.
// (These figures are of replayed graphs on a card that has not heated up.  Among other calls the card is at its 1,000 W and the clock
// falls: 32 x 16,384 takes 298 us there, 16 x 8,192 with trees of 64 360.)
// P is rounded to bfloat16 for the product, the sum it is divided by is not: beside the formula in 64 bits a result is off by 0.0023 of
// its size, of which its own rounding is 0.0017.
// Of a tile's values only the 16 keys at a time that hold a valid one are multiplied; rows behind the last valid one (stale
// places of a page, other requests' tokens) are set to zero first, for 0 * NaN is NaN.  Where a tile's keys are not seen by
// all rows alike (the step's own tokens, a window's edge) values that are not finite are taken out of the product and added
// by hand to the rows that see them.  (In units of 256 rows both sets do that in the tile that they share, and write the same bytes.)
// Every mbarrier wait is bounded (status codes 41..45, see attention_tc.cu).  No cluster multicast.
#include "attention_tc.cuh"
#include "tree_attention.cuh"
#include <math_constants.h>

#include <type_traits>

namespace pmm {

constexpr int kTtSeqs = 1024;  // requests whose lengths fit shared memory
constexpr int kTtRows = 128;   // rows of a set
constexpr int kTtThreads = 12 * 32;  // copies, two warps that issue, one without work, two sets of four
// tensor memory: S (and P) of the two sets of warps, O of the two
constexpr unsigned kTtO = 256, kTtCols = 512;
__host__ __device__ constexpr int tree_q_sub() { return kTtRows * kAtDhBlock * 2; }        // a sub-tile of Q: 64 head-size columns
// Tiles in flight (16 or 32 KB each): what queries and lengths leave of shared memory (32 x 16,384: 245 us with 5, 260 with 4).  K_j is copy
// 2 j, V_j copy 2 j + 3 of the block (the order in which they are asked for; there is no copy 1), in slot (copy % ring).  A copy's barrier
// tells it only from the one before on that barrier, and a wait that skips one may take the last but one for its own; so there are
// as many barriers as make all copies of one to be of one kind and, where the sets take the tiles in turn, of one set.
__host__ __device__ constexpr int tree_ring(int dh, bool wide) { return dh == 64 ? 11 : wide ? 4 : 5; }
__host__ __device__ constexpr int tree_bars(int ring) { return ring % 4 == 0 ? ring : 4 * ring; }
__host__ __device__ constexpr size_t tree_smem(int dh, bool wide) {
  return static_cast<size_t>(dh / kAtDhBlock) * ((wide ? 2 : 1) * tree_q_sub() + tree_ring(dh, wide) * kAtKvSub) + 1024 /*alignment*/;
}

// S = Q K^T: both K-major; O += P V: V as it lies in the cache (MN-major), all DH columns at once.
constexpr int kTtHalf = kAtKeys / 2;  // keys of an S product
constexpr unsigned kTtIdescS = (1u << 4) | (1u << 7) | (1u << 10) | (static_cast<unsigned>(kTtHalf >> 3) << 17) | (static_cast<unsigned>(kTtRows >> 4) << 24);
__host__ __device__ constexpr unsigned tree_idesc_o(int dh) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | (static_cast<unsigned>(dh >> 3) << 17) | (static_cast<unsigned>(kTtRows >> 4) << 24);
}
// Products and commits by one elected thread of a warp that is here as a whole, the same one every time.  elect.sync is how the
// compiler learns that a single thread issues: a commit takes 8 clocks, with a predicate (lane == 0) 55, and eight products 312 or
// fewer, not 401.
__device__ __forceinline__ void tree_mma_ss(unsigned tmem_d, unsigned long long a_desc, unsigned long long b_desc, unsigned idesc, unsigned accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, l;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "elect.sync _|l, 0xffffffff;\n\t"
      "@l tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n"
      :
      : "r"(tmem_d), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// (the A operand in tensor memory: row i in lane i, two neighbouring elements a column)
__device__ __forceinline__ void tree_mma_ts(unsigned tmem_d, unsigned tmem_a, unsigned long long b_desc, unsigned idesc, unsigned accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, l;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "elect.sync _|l, 0xffffffff;\n\t"
      "@l tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n"
      :
      : "r"(tmem_d), "r"(tmem_a), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tree_commit(unsigned long long* bar) {
  asm volatile(
      "{\n\t.reg .pred l;\n\t"
      "elect.sync _|l, 0xffffffff;\n\t"
      "@l tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(smem_u32(bar))
      : "memory");
}

// 16 bytes to shared memory, or zeros.
__device__ __forceinline__ void cp_async16_fill(void* dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(smem_u32(dst)), "l"(src), "r"(there ? 16 : 0) : "memory");
}

// 32 lanes of tensor memory x 16 columns, a lane a row.
__device__ __forceinline__ void tree_tmem_ld16(unsigned taddr, unsigned* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tree_tmem_st16(unsigned taddr, const unsigned* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};\n"
      :
      : "r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// Tensor maps, two-dimensional with boxes of 64 columns: the pool's rows, the step's keys and values.
struct TreeMaps {
  CUtensorMap pool, own_k, own_v;
};
struct TreeTcArgs {
  const bf16* q;
  long long ldq;
  const bf16* v;        // the step's values, for values that are not finite
  long long ldv;
  const bf16* pool;
  const int* block_table;
  int max_blocks, pages;
  const int* held;
  const int* cu;
  const int* positions;
  const unsigned long long* mask;
  int words;
  const float* sink;
  bf16* out;
  float4* part_o;       // [2 * blocks][DH / 4][rows]: neighbouring threads, a row each, write neighbouring places
  float2* part_ml;      // [2 * blocks][rows]
  int* cuts;            // [blocks][8]: a unit that shares cut: its rows (0: none), first token, head, row tile, last block
  float scale_log2;
  int window;
  int window_step;      // the window limits the step's own tokens too, by their positions
  int page_size, box, n_seq, T, Hq, Hkv, shares;
  int rows;             // of a unit: 128 or 256
  int* status;
};

// One request as the walk sees it.
struct TreeSeq {
  int t0, n_new, held, first;  // first: the cached key at which its tiles begin
  int n_rt, ctx_tiles, nt;     // row tiles of a key/value head, tiles of cached keys, tiles of a unit
};
__device__ __forceinline__ TreeSeq tree_seq(const TreeTcArgs& a, int t0, int t1, int held, int first) {
  TreeSeq s;
  s.t0 = t0;
  s.n_new = t1 - t0;
  s.held = held;
  s.first = first;
  const int G = a.Hq / a.Hkv;
  s.n_rt = (s.n_new * G + a.rows - 1) / a.rows;
  s.ctx_tiles = held > first ? (held - first + kAtKeys - 1) / kAtKeys : 0;
  s.nt = s.ctx_tiles + (s.n_new + kAtKeys - 1) / kAtKeys;
  return s;
}

// The lengths of all requests in shared memory, and the running sum of their tiles.  The order of the units: where all requests have as
// many row tiles, row tile by row tile over all requests, so that the blocks that read the same keys do so at the same time
// (one behind the other every row tile brought them from memory anew: the wide trees' 0.6 GB became 2.1); else request by request.
struct TreePlan {
  int* pre;    // [n_seq + 1] tiles in front of a request, in the first row tile's round or in all
  int* cu;     // [n_seq + 1]
  int* held;   // [n_seq]
  int* first;  // [n_seq]
  int rounds;  // row tiles of every request, or 0: requests differ
  int total;
};
__host__ __device__ constexpr size_t tree_plan_bytes(int n_seq) { return (4 * static_cast<size_t>(n_seq) + 2) * sizeof(int); }

// Called by all THREADS threads of the block; red: shared memory for 32 ints.
template <int THREADS>
__device__ __forceinline__ void tree_plan(const TreeTcArgs& a, TreePlan& p, int* red) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) red[31] = 0;
  __syncthreads();
  int same = -1;
  bool differ = false;
  for (int s = tid; s < a.n_seq; s += THREADS) {
    const int t0 = min(max(a.cu[s], 0), a.T), t1 = min(max(a.cu[s + 1], t0), a.T);
    const int held = max(0, static_cast<int>(min(static_cast<long long>(a.held[s]), static_cast<long long>(a.max_blocks) * a.page_size)));
    int first = 0;
    if (a.window != 0) {  // the first key that any of the request's tokens may see
      int pos = 0x7fffffff;
      for (int t = t0; t < t1; ++t) pos = min(pos, a.positions[t]);
      first = t1 > t0 ? min(first_visible(pos, a.window), held) / a.box * a.box : 0;
    }
    p.cu[s] = t0;
    if (s == a.n_seq - 1) p.cu[s + 1] = t1;
    p.held[s] = held;
    p.first[s] = first;
    const int n_rt = tree_seq(a, t0, t1, held, first).n_rt;
    if (n_rt > 0) {
      differ |= same > 0 && n_rt != same;
      same = n_rt;
    }
  }
  if (same > 0) atomicMax(&red[31], same);
  const int any_differs = __syncthreads_or(differ);
  const int most = red[31];
  p.rounds = __syncthreads_or(any_differs || (same > 0 && same != most)) ? 0 : most;
  int total = 0;
  for (int base = 0; base < a.n_seq; base += THREADS) {
    const int s = base + tid;
    int tiles = 0;
    if (s < a.n_seq) {
      const TreeSeq q = tree_seq(a, p.cu[s], p.cu[s + 1], p.held[s], p.first[s]);
      tiles = q.n_rt > 0 ? q.nt * a.Hkv * (p.rounds > 0 ? 1 : q.n_rt) : 0;
    }
    int run = tiles;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += up;
    }
    if (lane == 31) red[warp] = run;
    __syncthreads();
    int before = total;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
      if (w < warp) before += red[w];
      total += red[w];
    }
    if (s < a.n_seq) p.pre[s] = before + run - tiles;
    __syncthreads();
  }
  if (tid == 0) p.pre[a.n_seq] = total;
  __syncthreads();
  p.total = total * max(p.rounds, 1);
}

// How many blocks share `total` tiles, the tile at which block b's share begins, and the block in whose share tile x lies.
__device__ __forceinline__ int tree_shares(const TreeTcArgs& a, int total) { return max(1, min(a.shares, total)); }
__device__ __forceinline__ int tree_begin(int b, int total, int shares) { return static_cast<int>(static_cast<long long>(b) * total / shares); }
__device__ __forceinline__ int tree_block(int x, int total, int shares) {
  return static_cast<int>(((static_cast<long long>(x) + 1) * shares - 1) / total);
}

// A stretch of one unit's tiles.
struct TreeSeg {
  TreeSeq s;
  int seq, hk, rt;       // request, key/value head, row tile
  int unit;              // the unit's first tile, counted over all
  int j0, j1;            // the stretch's tiles within the unit
};
// The stretch that begins at tile `at` and ends with its unit or at `end`.
__device__ __forceinline__ TreeSeg tree_seg(const TreeTcArgs& a, const TreePlan& p, int at, int end) {
  const int round = p.pre[a.n_seq], rt = p.rounds > 0 ? at / round : 0, in_round = at - rt * round;
  int lo = 0, hi = a.n_seq - 1;  // the last request that begins at or before (behind requests without tiles)
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (p.pre[mid] <= in_round)
      lo = mid;
    else
      hi = mid - 1;
  }
  TreeSeg g;
  g.seq = lo;
  g.s = tree_seq(a, p.cu[lo], p.cu[lo + 1], p.held[lo], p.first[lo]);
  const int off = in_round - p.pre[lo], u = off / g.s.nt;
  if (p.rounds > 0) {
    g.hk = u;
    g.rt = rt;
  } else {
    g.hk = u / g.s.n_rt;
    g.rt = u - g.hk * g.s.n_rt;
  }
  g.unit = at - (off - u * g.s.nt);
  g.j0 = at - g.unit;
  g.j1 = min(g.s.nt, end - g.unit);
  return g;
}
// Valid keys of tile j.
__device__ __forceinline__ int tree_valid(const TreeSeq& s, int j) {
  return j < s.ctx_tiles ? min(kAtKeys, s.held - s.first - j * kAtKeys) : min(kAtKeys, s.n_new - (j - s.ctx_tiles) * kAtKeys);
}

template <int DH, bool WIDE>
__global__ void __launch_bounds__(kTtThreads, 1) tree_attention_tc_kernel(const __grid_constant__ TreeMaps maps, const __grid_constant__ TreeTcArgs a) {
  constexpr int NSUB = DH / kAtDhBlock;
  constexpr int kRing = tree_ring(DH, WIDE), kBars = tree_bars(kRing);
  constexpr int kRows = WIDE ? 2 * kTtRows : kTtRows;  // of a unit
  constexpr int kSlot = NSUB * kAtKvSub;
  constexpr int kQSub = tree_q_sub();
  extern __shared__ unsigned char smem_raw[];
  // the queries are in place / have been read by a unit's last S; a slot is full / empty; a set's S and P are there; a unit's last
  // products are done; both sets' maxima and sums are there; both have read their O
  __shared__ __align__(8) unsigned long long bar_q, bar_qfree, bar_full[kBars], bar_empty[kRing], bar_s[2][2], bar_p[2][2], bar_o[2], bar_done, bar_ml, bar_read;
  __shared__ float2 s_ml[2][2][kTtRows];  // (of two stretches in turn: one set may be a stretch ahead)
  __shared__ unsigned s_tmem_base;
  __shared__ int s_abort, s_red[32], s_bad[2];

  unsigned char* sQ = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* sRing = sQ + (WIDE ? 2 : 1) * NSUB * kQSub;
  TreePlan plan;
  plan.pre = reinterpret_cast<int*>(sRing + kRing * kSlot);
  plan.cu = plan.pre + a.n_seq + 1;
  plan.held = plan.cu + a.n_seq + 1;
  plan.first = plan.held + a.n_seq;

  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const int G = a.Hq / a.Hkv;
  if (tid == 0) {
    mbar_init(&bar_q, 8);
    mbar_init(&bar_qfree, 2);
    for (int i = 0; i < kBars; ++i) mbar_init(&bar_full[i], 1);
    for (int i = 0; i < kRing; ++i) mbar_init(&bar_empty[i], WIDE ? 2 : 1);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar_o[i], 1);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        mbar_init(&bar_s[i][h], 1);
        mbar_init(&bar_p[i][h], 4);
      }
    }
    mbar_init(&bar_done, 2);
    mbar_init(&bar_ml, 8);
    mbar_init(&bar_read, 8);
    mbar_arrive(&bar_full[1]);  // (copy 1, which is none, has come and gone)
    for (int i = 0; i < (WIDE ? 2 : 1); ++i) mbar_arrive(&bar_empty[1]);
    s_abort = 0;
    s_bad[0] = s_bad[1] = -1;
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    asm volatile("prefetch.tensormap [%0];\n" ::"l"(reinterpret_cast<unsigned long long>(&maps.pool)) : "memory");
  }
  pdl_wait();
  pdl_launch_dependents();  // (behind the wait: the merge's blocks would hold places that the launch in front needs)
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(&s_tmem_base)), "r"(kTtCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
  tree_plan<kTtThreads>(a, plan, s_red);
  asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
  const unsigned tmem_base = s_tmem_base;
  const int total = plan.total;
  const int shares = tree_shares(a, total);
  int* record = a.cuts + 8 * blockIdx.x;  // of the unit that is cut at this block's first tile, for the merge
  if (static_cast<int>(blockIdx.x) >= shares || total == 0) {
    if (tid == 0) record[0] = 0;
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem_base), "r"(kTtCols) : "memory");
    return;
  }
  const int begin = tree_begin(blockIdx.x, total, shares), end = tree_begin(blockIdx.x + 1, total, shares);
  const int n_tiles = end - begin;  // (at least one)
  volatile int* abort_flag = &s_abort;
  auto give_up = [&](int code) {
    if (!*abort_flag) atomicExch(a.status, code);
    s_abort = 1;
  };

  if (warp == 0) {
    // ---------------------------------------------------------------- TMA producer (the whole warp walks, a lane a box)
    const int page_size = a.page_size;
    const int per = kAtKeys / a.box;  // boxes of a tile of cached keys
    int n_k = 0, n_v = 0;             // copies requested
    bool ok = true;
    struct Tile {
      int row, valid, hk;  // row of the pool (of k and v) at which this lane's box begins, keys of the tile
      bool own;            // the step's own tokens
    };
    auto request = [&](const Tile& t, bool is_v) {
      const int item = is_v ? 2 * n_v + 3 : 2 * n_k, slot = item % kRing;
      if (item >= kRing && ok) {
        int got = 1;
        if (lane == 0) got = mbar_wait(&bar_empty[slot], (item / kRing - 1) & 1, abort_flag) ? 1 : 0;
        ok = __shfl_sync(0xffffffffu, got, 0) != 0;
        if (!ok && lane == 0) give_up(42);
      }
      if (!ok) return;
      const int keys = t.own ? kAtBox : a.box;  // of a box
      const int boxes = (t.valid + keys - 1) / keys;
      unsigned long long* full = &bar_full[item % kBars];
      if (lane == 0) mbar_expect_tx(full, static_cast<unsigned>(boxes * keys * NSUB * 128));
      __syncwarp();
      const int d = lane % NSUB, b = lane / NSUB;  // a lane a copy: sub-tile of 64 columns, box
      const int row = __shfl_sync(0xffffffffu, t.row, b);
      if (b < boxes)
        tma_load_2d(sRing + slot * kSlot + d * kAtKvSub + b * keys * 128, t.own ? (is_v ? &maps.own_v : &maps.own_k) : &maps.pool,
                    t.hk * DH + d * kAtDhBlock, row + (is_v && !t.own ? page_size : 0), full);
      ++(is_v ? n_v : n_k);
    };
    Tile prev{};
    for (int at = begin; at < end && ok;) {
      const TreeSeg g = tree_seg(a, plan, at, end);
      const int* bt = a.block_table + static_cast<size_t>(g.seq) * a.max_blocks;
      int batch = g.j0 * per - 32, batch_row = 0;  // a lane's box of the 32 whose rows are at hand
      for (int j = g.j0; j < g.j1 && ok; ++j, ++at) {
        Tile t;
        t.valid = tree_valid(g.s, j);
        t.hk = g.hk;
        t.own = j >= g.s.ctx_tiles;
        if (!t.own) {
          if (j * per >= batch + 32) {
            batch = j * per;
            const int key = g.s.first + (batch + lane) * a.box;
            batch_row = 0;
            if (key < g.s.held) {
              const int page = min(max(bt[key / page_size], 0), a.pages - 1);  // (no read leaves the pool)
              batch_row = page * 2 * page_size + key % page_size;
            }
          }
          t.row = __shfl_sync(0xffffffffu, batch_row, (j * per - batch + lane) & 31);
        } else {
          t.row = g.s.t0 + (j - g.s.ctx_tiles) * kAtKeys + lane * kAtBox;
        }
        request(t, false);
        if (at > begin && ok) request(prev, true);
        prev = t;
      }
    }
    if (ok) request(prev, true);
    __syncwarp();
    if (lane == 0 && s_abort) {
      // copies already requested still write into this block's shared memory: wait for them
      const int items = 2 * max(n_k, n_v) + 3;
      for (int u = 0; u < kRing; ++u) {  // the last copy of every slot
        int it = items - 1;
        while (it >= 0 && (it % kRing != u || ((it & 1) ? it == 1 || (it - 3) / 2 >= n_v : it / 2 >= n_k))) --it;
        if (it < 0) continue;
        for (unsigned i = 0; i < kSpinLimit && !mbar_try_wait(&bar_full[it % kBars], (it / kBars) & 1); ++i) {
        }
      }
    }
  } else if (warp == 1 || warp == 2) {
    // ---------------------------------------------------------------- MMA issuers, one a set (the whole warp walks, one lane issues)
    const int set = warp - 1;
    // What the products are issued with, and everything that decides whether they are, comes out of a reduction or a vote: it is known to
    // be the same in the whole warp and stays in uniform registers (130 to 180 clocks a product where it is not, 64 where it is).
    auto uniform = [](unsigned x) { return static_cast<int>(__reduce_max_sync(0xffffffffu, x)); };
    const int n = uniform(n_tiles);
    const unsigned tmem = uniform(tmem_base), s_tmem = tmem + kAtKeys * set, o_tmem = tmem + kTtO + 128 * set;
    const unsigned long long q_desc = umma_desc(sQ + (WIDE ? set * NSUB * kQSub : 0)), ring_desc = umma_desc(sRing);
    // (of a V tile: 64 columns further lie one sub-tile further)
    const unsigned long long v_ring = (ring_desc & ~(0x3fffull << 16)) | (static_cast<unsigned long long>(kAtKvSub >> 4) << 16);
    auto wait = [&](unsigned long long* bar, unsigned parity) {
      return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag)) != 0;  // (no lane may fall a phase behind)
    };
    constexpr int kStep = WIDE ? 1 : 2;
    // The set's tiles, stretch by stretch.  Two walks over them: of the S products and, a tile behind, of the P V.  (A set has tiles in
    // every stretch but those of one tile, and no two of those without one follow one another.)  Tiles are counted within the block.
    struct Walk {
      int seg, t, end;               // the stretch's number, the next tile, the stretch's end
      int h;                         // the next half of it
      int live, in, rows;            // in: its queries are in place; rows: the set has some (of 256, the second may have none)
      int own, last;                 // the unit's first tile of the step's own tokens, its last tile
      int ctx_steps, last_steps;     // sixteens of keys in the last tile of cached keys, and in the last of all
      int slot, bar, phase;          // of the tile's copy
    };
    auto load = [&](Walk& w, int at) {
      const TreeSeg g = tree_seg(a, plan, at, end);
      w.end = uniform(g.unit + g.j1 - begin);
      w.rows = uniform(!WIDE || g.s.n_new * G - g.rt * kRows > set * kTtRows ? 1u : 0u);
      // (negative where the unit began in an earlier block: moved up by 2^30 to be compared as unsigned)
      w.own = uniform(g.unit + g.s.ctx_tiles - begin + (1 << 30)) - (1 << 30);
      w.last = uniform(g.unit + g.s.nt - 1 - begin + (1 << 30)) - (1 << 30);
      w.ctx_steps = uniform(g.s.ctx_tiles > 0 ? (tree_valid(g.s, g.s.ctx_tiles - 1) + 15) / 16 : 0);
      w.last_steps = uniform((tree_valid(g.s, g.s.nt - 1) + 15) / 16);
    };
    auto leave = [&](Walk& w) {
      w.in = 0;
      w.live = w.end < n;
      if (w.live) {
        load(w, begin + w.end);
        ++w.seg;
      }
    };
    auto next = [&](Walk& w) {  // the set's next tile
      w.t += kStep;
      w.slot += 2 * kStep;
      w.slot = w.slot >= kRing ? w.slot - kRing : w.slot;
      w.bar += 2 * kStep;
      w.phase = w.bar >= kBars ? w.phase ^ 1 : w.phase;
      w.bar = w.bar >= kBars ? w.bar - kBars : w.bar;
    };
    Walk ws, wp;
    ws.seg = ws.in = 0;
    ws.t = WIDE ? 0 : set;
    ws.h = 0;
    ws.live = 1;
    ws.slot = ws.bar = WIDE ? 0 : 2 * set;  // (copy 2 t)
    ws.phase = 0;
    load(ws, begin);
    wp = ws;
    const int first_v = 2 * wp.t + 3;       // (copy 2 t + 3)
    wp.slot = first_v % kRing;
    wp.bar = first_v % kBars;
    wp.phase = first_v / kBars & 1;
    auto steps_of = [](const Walk& w) { return w.t == w.own - 1 ? w.ctx_steps : w.t == w.last ? w.last_steps : kAtKeys / 16; };
    auto full = [&](const Walk& w) { return wait(&bar_full[w.bar], w.phase); };
    // a slot's copy has been used (by a set without rows, at once)
    auto used = [&](const Walk& w) {
      if (w.rows)
        tree_commit(&bar_empty[w.slot]);
      else if (lane == 0)
        mbar_arrive(&bar_empty[w.slot]);
    };
    auto product_s = [&](const Walk& w, int h) {
      asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
      const unsigned long long k_desc = ring_desc + static_cast<unsigned>(w.slot * (kSlot >> 4) + h * (kTtHalf * 128 >> 4));
#pragma unroll
      for (int k = 0; k < DH / 16; ++k)
        tree_mma_ss(s_tmem + kTtHalf * h, q_desc + (k >> 2) * (kQSub >> 4) + 2 * (k & 3), k_desc + (k >> 2) * (kAtKvSub >> 4) + 2 * (k & 3), kTtIdescS,
                    k > 0 ? 1u : 0u);
      tree_commit(&bar_s[set][h]);
    };
    auto product_o = [&](const Walk& w, int h, int sixteens, int more) {
      asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
      const unsigned long long v_desc = v_ring + static_cast<unsigned>(w.slot * (kSlot >> 4) + h * (kTtHalf * 128 >> 4));
      auto product = [&](int k) {  // 16 keys: 16 rows of 128 bytes of every sub-tile
        tree_mma_ts(o_tmem, s_tmem + kTtHalf * h + 8 * k, v_desc + ((k * 16 * 128) >> 4), tree_idesc_o(DH), k > 0 ? 1u : static_cast<unsigned>(more));
      };
      if (sixteens == 4) {
#pragma unroll
        for (int k = 0; k < 4; ++k) product(k);
      } else {
        for (int k = 0; k < sixteens; ++k) product(k);
      }
      tree_commit(&bar_o[set]);
    };
    int taken = 0;  // bit h: the place of half h holds an S or P that has not been used
    // Every next S whose place is free; another stretch's once all products of this one have been issued (its queries wait for what waits for them).
    auto issue_s = [&]() {
      while (ws.live) {
        if (!ws.in) {
          if (taken) return true;
          if (!wait(&bar_q, ws.seg & 1)) return false;
          ws.in = 1;
        }
        if (ws.t >= ws.end) {  // the set's last of the stretch, or none in it: its queries may make way
          tree_commit(&bar_qfree);
          leave(ws);
          continue;
        }
        if (taken >> ws.h & 1) return true;
        if (ws.h == 0 && !full(ws)) return false;
        if (ws.rows) product_s(ws, ws.h);
        taken |= 1 << ws.h;
        if (ws.h == 0 && steps_of(ws) > 4) {
          ws.h = 1;
        } else {
          used(ws);
          ws.h = 0;
          next(ws);
        }
      }
      return true;
    };
    int code = issue_s() ? 0 : 43, n_p = 0;  // bit h: the parity of the next P of half h
    int more = 0, told = 0;                  // O goes on; the stretch's end has been told
    while (code == 0 && wp.live) {
      if (wp.t >= wp.end) {
        if (!told) tree_commit(&bar_done);
        told = more = 0;
        const int left = wp.seg;
        leave(wp);
        if (wp.live && !wait(&bar_read, left & 1)) code = 44;  // (its O has been read)
        continue;
      }
      // Whole tiles with another of the stretch behind them, both halves of their S made: the same without questions (a warp's way
      // through branches costs more than the products that it issues: 338 us with them where 305 without).
      if (ws.rows && taken == 3 && ws.in && ws.seg == wp.seg && ws.t == wp.t + kStep) {
        int until = wp.end;  // the first tile that is not whole, or the end
        if (wp.ctx_steps < 8 && wp.t < wp.own) until = min(until, wp.own - 1);
        if (wp.last_steps < 8) until = min(until, wp.last);
        for (; ws.t < until && code == 0;) {
          if (!full(wp) || !wait(&bar_p[set][0], n_p & 1)) {
            code = 44;
            break;
          }
          product_o(wp, 0, 4, more);
          more = 1;
          if (!full(ws)) {
            code = 43;
            break;
          }
          product_s(ws, 0);
          if (!wait(&bar_p[set][1], n_p >> 1)) {
            code = 44;
            break;
          }
          product_o(wp, 1, 4, 1);
          tree_commit(&bar_empty[wp.slot]);
          product_s(ws, 1);
          tree_commit(&bar_empty[ws.slot]);
          n_p ^= 3;
          next(wp);
          next(ws);
        }
        if (code != 0) break;
        if (!issue_s()) {  // (the stretch's queries may make way)
          code = 43;
          break;
        }
      }
      const int steps = steps_of(wp);
      if (!full(wp)) {
        code = 44;
        break;
      }
#pragma unroll 1
      for (int h = 0; h < (steps > 4 ? 2 : 1); ++h) {
        if (wp.rows) {
          if (!wait(&bar_p[set][h], n_p >> h & 1)) {
            code = 44;
            break;
          }
          n_p ^= 1 << h;
          product_o(wp, h, min(4, steps - 4 * h), more);
        }
        taken &= ~(1 << h);
        more = 1;
        if (h == 1 || steps <= 4) {
          used(wp);
          next(wp);
          if (wp.t >= wp.end) {
            tree_commit(&bar_done);
            told = 1;
          }
        }
        if (!issue_s()) {
          code = 43;
          break;
        }
      }
    }
    if (code != 0) give_up(code);
  } else if (warp >= 4) {
    // ---------------------------------------------------------------- softmax and output (a thread a row, two sets of warps)
    const int set = (warp - 4) >> 2, quarter = warp & 3;
    const int row = (WIDE ? set * kTtRows : 0) + quarter * 32 + lane;  // of the unit (quarter * 32 + lane: its lane of tensor memory)
    const unsigned lane_base = tmem_base + (static_cast<unsigned>(quarter * 32) << 16);
    const unsigned s_tmem = lane_base + kAtKeys * set, o_tmem = lane_base + kTtO + 128 * set;
    const int soft_tid = tid - 128, set_tid = soft_tid & 127;  // among the softmax threads, the set's
    bool alive = true;
    auto wait = [&](unsigned long long* bar, unsigned parity) {
      const bool got = __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag));
      if (!got) {
        if (lane == 0) give_up(45);
        alive = false;
      }
      return got;
    };
    // the stretch's query rows -> shared memory, swizzled (rows beyond the unit are zero)
    auto queries = [&](const TreeSeg& g) {
      const int n_rows = min(kRows, g.s.n_new * G - g.rt * kRows);
      constexpr int kPieces = DH / 8;
#pragma unroll 4
      for (int p = soft_tid; p < kRows * kPieces; p += 256) {  // neighbouring lanes take neighbouring pieces
        const int r = p / kPieces, c = p % kPieces, gr = g.rt * kRows + r, tk = gr / G;
        const bf16* src = r < n_rows ? a.q + (g.s.t0 + tk) * a.ldq + (g.hk * G + (gr - tk * G)) * DH + c * 8 : a.q;
        cp_async16_fill(sQ + ((r >> 7) * NSUB + (c >> 3)) * kQSub + at_swizzled(r & 127, c & 7), src, r < n_rows);
      }
      asm volatile("cp.async.wait_all;\n" ::: "memory");
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar_q);
    };
    int n_s = 0, n_half = 0;                              // bit h: the parity of the next S of half h; halves that this set has taken
    TreeSeg g = tree_seg(a, plan, begin, end);
    queries(g);
    if (soft_tid == 0) {  // (the block behind the one in which the unit begins tells the merge)
      const bool cut = g.j0 > 0 && g.unit >= tree_begin(blockIdx.x - 1, total, shares);
      record[0] = cut ? min(kRows, g.s.n_new * G - g.rt * kRows) : 0;
      record[1] = g.s.t0;
      record[2] = g.hk;
      record[3] = g.rt;
      record[4] = tree_block(g.unit + g.s.nt - 1, total, shares);
    }
    for (int seg = 0, at = begin; at < end && alive; ++seg) {
      const int n_rows = min(kRows, g.s.n_new * G - g.rt * kRows);
      const bool idle = (WIDE ? set * kTtRows : 0) + quarter * 32 >= n_rows;           // (the whole warp: none of its rows exists)
      const int my_tok = row < n_rows ? (g.rt * kRows + row) / G : 0;   // the row's token, of the request
      const int my_lo = a.window != 0 ? first_visible(a.positions[g.s.t0 + my_tok], a.window) : 0;  // its first cached key
      float m_run = -CUDART_INF_F, l_run = 0.f;           // maximum in use (exponent's unit), sum against it
      int edge = 0;                                       // behind it every row of the unit sees all cached keys
      if (a.window != 0) {
        const int last = (g.rt * kRows + n_rows - 1) / G;
        for (int tk = g.rt * kRows / G + lane; tk <= last; tk += 32) edge = max(edge, first_visible(a.positions[g.s.t0 + tk], a.window));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) edge = max(edge, __shfl_xor_sync(0xffffffffu, edge, o));
      }
      // whether the rows may see tile j's keys differently: the step's own tokens, and in front of the windows' last edge
      auto mixed = [&](const TreeSeg& of, int j) { return j >= of.s.ctx_tiles || of.s.first + j * kAtKeys < edge; };
      // the set's tiles: all of them, where it has rows, or every second, over all units
      const int first = WIDE ? (n_rows > set * kTtRows ? at : g.unit + g.j1) : at + ((at - begin + set) & 1);
      for (int t = first; t < g.unit + g.j1; t += WIDE ? 1 : 2) {
        const int j = t - g.unit, gt = t - begin;         // within the unit, of the block
        const bool own = j >= g.s.ctx_tiles;
        const int base = g.s.first + j * kAtKeys;         // (cached keys)
        const int valid = tree_valid(g.s, j);
        if (!wait(&bar_s[set][0], n_s & 1)) break;
        asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
        if (valid % 16 != 0 || mixed(g, j)) {
          // values that must not meet a probability of zero: rows behind the last valid one become zero; where rows see the
          // keys differently, so do values that are not finite
          const int item = 2 * gt + 3, slot = item % kRing;
          if (!wait(&bar_full[item % kBars], (item / kBars) & 1)) break;
          unsigned char* sV = sRing + slot * kSlot;
          const int from = mixed(g, j) ? 0 : valid * (DH / 8), to = (valid + 15) / 16 * 16 * (DH / 8);
          for (int p = from + set_tid; p < to; p += 128) {
            const int r = p / (DH / 8), c = p % (DH / 8);
            uint4* at16 = reinterpret_cast<uint4*>(sV + (c >> 3) * kAtKvSub + at_swizzled(r, c & 7));
            if (r >= valid) {
              *at16 = make_uint4(0u, 0u, 0u, 0u);
            } else {
              uint4 x = *at16;
              unsigned* w = reinterpret_cast<unsigned*>(&x);
              bool bad = false;
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                if ((w[e] & 0x7f80u) == 0x7f80u) {
                  w[e] &= 0xffff0000u;
                  bad = true;
                }
                if ((w[e] & 0x7f800000u) == 0x7f800000u) {
                  w[e] &= 0x0000ffffu;
                  bad = true;
                }
              }
              if (bad) {
                *at16 = x;
                reinterpret_cast<volatile int*>(s_bad)[seg & 1] = seg;
              }
            }
          }
          fence_proxy_async();
        }
        // Half h of the scores to probabilities; masked: some rows may not see some of the keys.
        auto half = [&](int h, auto masked) {
          const unsigned here = s_tmem + kTtHalf * h;
          unsigned long long w = 0ull;  // the bits of the row's visible keys among these 64
          if (decltype(masked)::value) {
            const int left = valid - kTtHalf * h;
            w = left >= 64 ? ~0ull : (1ull << left) - 1ull;
            if (own) {  // of its mask, or up to the token itself
              const int k0 = (j - g.s.ctx_tiles) * kAtKeys + kTtHalf * h, upto = my_tok + 1 - k0;
              if (a.mask)
                w &= k0 / 64 < a.words ? a.mask[static_cast<size_t>(g.s.t0 + my_tok) * a.words + k0 / 64] : 0ull;
              else
                w &= upto <= 0 ? 0ull : upto >= 64 ? ~0ull : (1ull << upto) - 1ull;
              if (a.window_step)  // (a place is one token for the whole warp)
                for (int i = 0; i < min(left, 64); ++i) w &= ~(static_cast<unsigned long long>(a.positions[g.s.t0 + k0 + i] < my_lo) << i);
            } else {
              const int skip = my_lo - (base + kTtHalf * h);
              w &= skip <= 0 ? ~0ull : skip >= 64 ? 0ull : ~0ull << skip;
            }
          }
          unsigned v[kTtHalf];
#pragma unroll
          for (int c = 0; c < 2; ++c) tmem_ld32(here + 32 * c, v + 32 * c);
          asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
          if (decltype(masked)::value) {
#pragma unroll
            for (int i = 0; i < kTtHalf; ++i)
              if (!(static_cast<unsigned>(w >> (i & 32)) >> (i & 31) & 1u)) v[i] = __float_as_uint(-CUDART_INF_F);
          }
          float mx[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) mx[u] = fmaxf(__uint_as_float(v[u]), __uint_as_float(v[u + 4]));
#pragma unroll
          for (int i = 8; i < kTtHalf; i += 8)
#pragma unroll
            for (int u = 0; u < 4; ++u) mx[u] = at_max3(mx[u], __uint_as_float(v[i + u]), __uint_as_float(v[i + u + 4]));
          const float m = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.scale_log2;  // scale > 0
          // raise the maximum in use only when the row's maximum has run ahead of it by more than kAtLazy
          const bool raise = (m > m_run + kAtLazy || m_run == -CUDART_INF_F) && m != -CUDART_INF_F;
          if (__any_sync(0xffffffffu, raise)) {
            const float alpha = raise ? at_ex2(m_run - m) : 1.f;
            m_run = raise ? m : m_run;
            l_run *= alpha;
            if (t > first || h == 1) {
              if (!wait(&bar_o[set], (n_half - 1) & 1)) return;  // this set's product before
              asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
#pragma unroll
              for (int c = 0; c < DH / 16; ++c) {
                unsigned o[16];
                tree_tmem_ld16(o_tmem + 16 * c, o);
                asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                tree_tmem_st16(o_tmem + 16 * c, o);
              }
            }
          }
          const float mu = m_run == -CUDART_INF_F ? 0.f : m_run;
          // P, two neighbouring keys a word, in the place of S
          float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int i = 0; i < kTtHalf / 2; ++i) {
            const float p0 = at_ex2(fmaf(__uint_as_float(v[2 * i]), a.scale_log2, -mu));  // masked: ex2(-inf) = 0
            const float p1 = at_ex2(fmaf(__uint_as_float(v[2 * i + 1]), a.scale_log2, -mu));
            sum[2 * (i & 1)] += p0;
            sum[2 * (i & 1) + 1] += p1;
            v[i] = at_pack(p0, p1);
          }
          tmem_st32(here, v);
          l_run += (sum[0] + sum[1]) + (sum[2] + sum[3]);
          asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
        };
        const bool plain = valid == kAtKeys && !mixed(g, j);
        const int halves = valid > kTtHalf ? 2 : 1;
#pragma unroll 1
        for (int h = 0; h < halves && alive; ++h) {
          if (h == 1) {
            if (!wait(&bar_s[set][1], n_s >> 1 & 1)) break;
            asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
          }
          n_s ^= 1 << h;
          if (!idle) {
            if (plain)
              half(h, std::false_type{});
            else
              half(h, std::true_type{});
          }
          ++n_half;
          asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
          __syncwarp();
          if (lane == 0) mbar_arrive(&bar_p[set][h]);
        }
        if (!alive) break;
      }
      if (!alive) break;
      const TreeSeg now = g;
      const int len = now.j1 - now.j0;                    // tiles of the stretch
      at += len;
      if (!WIDE) {
        s_ml[seg & 1][set][row] = make_float2(m_run, l_run);
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar_ml);
      }
      if (at < end) {  // the next stretch's queries, as soon as the last S of this one has been made
        g = tree_seg(a, plan, at, end);
        if (!wait(&bar_qfree, seg & 1)) break;
        queries(g);
      }

      // ---- the stretch's result once the last products have finished: of every set's rows, or the two sets' parts joined, half of the columns each
      if ((!WIDE && !wait(&bar_ml, seg & 1)) || !wait(&bar_done, seg & 1)) break;
      asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
      const bool whole = now.j0 == 0 && now.j1 == now.s.nt;
      const bool repair = reinterpret_cast<volatile int*>(s_bad)[seg & 1] == seg;
      if (!idle) {
        constexpr int kCols = WIDE ? DH : DH / 2;
        const int col0 = WIDE ? 0 : set * kCols;
        float m = m_run, l = l_run, w0 = 1.f, w1 = 1.f;   // maximum and sum, and what the two sets' parts are multiplied by
        if (!WIDE) {
          const float2 ml0 = s_ml[seg & 1][0][row], ml1 = s_ml[seg & 1][1][row];
          m = fmaxf(ml0.x, ml1.x);
          const float mu = m == -CUDART_INF_F ? 0.f : m;
          w0 = at_ex2(ml0.x - mu);                        // (a set that saw no key: 0)
          w1 = at_ex2(ml1.x - mu);
          l = ml0.y * w0 + ml1.y * w1;
        }
        const int gr = now.rt * kRows + row, tk = gr / G, hq = now.hk * G + (gr - tk * G);
        const bool row_ok = row < n_rows;
        if (whole) {
          if (a.sink != nullptr && row_ok) {
            // a score without key or value that counts once (of -inf: not at all); maxima are kept in units of log 2
            const float sk = a.sink[hq] * 1.4426950408889634f;
            const float m_new = fmaxf(m, sk), mu = m_new == -CUDART_INF_F ? 0.f : m_new, f = exp2f(m - mu);
            l = l * f + exp2f(sk - mu);
            w0 *= f;
            w1 *= f;
          }
          const float inv = l == 0.f ? 0.f : 1.f / l;     // (NaN stays NaN)
          w0 *= inv;
          w1 *= inv;
        }
        // whose parts: its own, or both sets' (of a single tile, of the one whose turn it was)
        const bool in0 = WIDE ? set == 0 : len > 1 || (((now.unit + now.j0 - begin) & 1) == 0), in1 = WIDE ? set == 1 : len > 1 || !in0;
        const size_t slot = 2 * static_cast<size_t>(blockIdx.x) + (now.j0 > 0 ? 0 : 1);
        float4* part = a.part_o + (slot * (DH / 4) + col0 / 4) * kRows + row;
        bf16* out = a.out + (static_cast<size_t>(now.s.t0 + tk) * a.Hq + hq) * DH + col0;
#pragma unroll
        for (int c = 0; c < kCols / 32; ++c) {
          float o[32];
          unsigned x[32];
          const unsigned from = lane_base + kTtO + col0 + 32 * c;
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0.f;
          __syncwarp();
          if (in0) {
            tmem_ld32(from, x);
            asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __uint_as_float(x[e]) * w0;
          }
          if (in1) {
            tmem_ld32(from + 128, x);
            asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = fmaf(__uint_as_float(x[e]), w1, o[e]);
          }
          if (repair) {
            // values that are not finite, to the rows that see their keys
            for (int j = now.j0; j < now.j1; ++j) {
              const bool own = j >= now.s.ctx_tiles;
              if (!mixed(now, j)) continue;
              const int valid = tree_valid(now.s, j);
              for (int k = 0; k < valid; ++k) {
                const bf16* vr;
                const int key = now.s.first + j * kAtKeys + k, node = (j - now.s.ctx_tiles) * kAtKeys + k;
                bool see;
                if (own) {
                  vr = a.v + (now.s.t0 + node) * a.ldv + now.hk * DH;
                  see = a.mask ? node < 64 * a.words && (a.mask[static_cast<size_t>(now.s.t0 + my_tok) * a.words + (node >> 6)] >> (node & 63) & 1ull)
                               : node <= my_tok;
                  see = see && (!a.window_step || a.positions[now.s.t0 + node] >= my_lo);
                } else {
                  const int page = min(max(a.block_table[static_cast<size_t>(now.seq) * a.max_blocks + key / a.page_size], 0), a.pages - 1);
                  vr = a.pool + ((static_cast<long long>(page) * 2 + 1) * a.page_size + key % a.page_size) * a.Hkv * DH + now.hk * DH;
                  see = key >= my_lo;
                }
                if (!see) continue;
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                  const float y = __bfloat162float(vr[col0 + 32 * c + e]);
                  if (!(fabsf(y) < CUDART_INF_F)) o[e] += y;
                }
              }
            }
          }
          if (row_ok && whole) {
#pragma unroll
            for (int e = 0; e < 32; e += 8)
              *reinterpret_cast<uint4*>(out + 32 * c + e) = make_uint4(at_pack(o[e], o[e + 1]), at_pack(o[e + 2], o[e + 3]), at_pack(o[e + 4], o[e + 5]),
                                                                      at_pack(o[e + 6], o[e + 7]));
          } else if (row_ok) {
#pragma unroll
            for (int e = 0; e < 32; e += 4) part[static_cast<size_t>(8 * c + e / 4) * kRows] = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
          }
        }
        if (!whole && row_ok && (WIDE || set == 0)) a.part_ml[slot * kRows + row] = make_float2(m, l);
      }
      asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar_read);
    }
  }

  asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
  __syncthreads();
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem_base), "r"(kTtCols) : "memory");
  }
}

// Units that the shares cut: block (x, y) takes the unit that block x + 1 of the launch in front has told, and the y-th piece of it.
//   M = max m_i;  o = sum_i o_i 2^(m_i - M) / sum_i l_i 2^(m_i - M)
// A warp takes 8 rows of 16 columns: 128 bytes of a part at a time and whole sectors of the result.
constexpr int kTmThreads = 256, kTmPieces = 16;

template <int DH>
__global__ void __launch_bounds__(kTmThreads) tree_merge_kernel(const __grid_constant__ TreeTcArgs a) {
  pdl_launch_dependents();
  pdl_wait();  // (every block waits: the next launch takes this one's end for that of both)
  const int share = blockIdx.x + 1;
  const int4 cut = *reinterpret_cast<const int4*>(a.cuts + 8 * share);
  const int n_rows = cut.x, t0 = cut.y, hk = cut.z, rt = cut.w;
  if (n_rows == 0) return;
  const int last = a.cuts[8 * share + 4];
  const int G = a.Hq / a.Hkv, lane = threadIdx.x & 31;
  constexpr int kBatch = 4;
  for (int i = blockIdx.y * (kTmThreads / 32) + threadIdx.x / 32; i < (n_rows + 7) / 8 * (DH / 16); i += kTmPieces * (kTmThreads / 32)) {
    const int r = i / (DH / 16) * 8 + (lane & 7), c4 = i % (DH / 16) * 4 + (lane >> 3);
    if (r >= n_rows) continue;
    const int row = rt * a.rows + r, tk = row / G, hq = hk * G + (row - tk * G);
    float mx = -CUDART_INF_F, sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    if (a.sink != nullptr) {
      mx = a.sink[hq] * 1.4426950408889634f;
      sum = 1.f;
    }
    for (int c0 = share - 1; c0 <= last; c0 += kBatch) {
      float2 ml[kBatch];
      float4 x[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int c = min(c0 + u, last);
        const size_t slot = 2 * static_cast<size_t>(c) + (c == share - 1 ? 1 : 0);  // the unit's beginning ends its block's share
        ml[u] = a.part_ml[slot * a.rows + r];
        x[u] = a.part_o[(slot * (DH / 4) + c4) * a.rows + r];
      }
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        if (c0 + u > last || ml[u].y == 0.f) continue;  // (a part in which the row sees no key)
        const float m_new = fmaxf(mx, ml[u].x);
        const float keep = mx == -CUDART_INF_F ? 0.f : exp2f(mx - m_new), w = exp2f(ml[u].x - m_new);
        acc.x = acc.x * keep + w * x[u].x;
        acc.y = acc.y * keep + w * x[u].y;
        acc.z = acc.z * keep + w * x[u].z;
        acc.w = acc.w * keep + w * x[u].w;
        sum = sum * keep + w * ml[u].y;
        mx = m_new;
      }
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    stf4(a.out + (static_cast<size_t>(t0 + tk) * a.Hq + hq) * DH + 4 * c4, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
  }
}

template <int DH, bool WIDE>
int launch_tree_tc(const TreeMaps& maps, const TreeTcArgs& a, cudaStream_t stream) {
  const size_t smem = tree_smem(DH, WIDE) + tree_plan_bytes(a.n_seq);
  auto kern = tree_attention_tc_kernel<DH, WIDE>;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));  // (of the current device: at every call)
  if (e != cudaSuccess) return static_cast<int>(e);
  launch_pdl(kern, dim3(a.shares), dim3(kTtThreads), smem, stream, maps, a);
  const int st = launch_status();
  if (st != 0 || a.shares == 1) return st;
  launch_pdl(tree_merge_kernel<DH>, dim3(a.shares - 1, kTmPieces), dim3(kTmThreads), 0, stream, a);
  return launch_status();
}

}  // namespace pmm

// Whether pmm_tree_attention_tc takes this shape.
static bool tree_tc_supported(int Hq, int Hkv, int Dh, int page_size, long long pages, int n_seq) {
  return Hq > 0 && Hkv > 0 && Hq % Hkv == 0 && (Dh == 64 || Dh == 128) && page_size > 0 && page_size % 8 == 0 && pages > 0 &&
         pages * 2 * page_size <= 0x7fffffffll && n_seq <= pmm::kTtSeqs;
}

// Floats of scratch for `sms` multiprocessors: two parts a block of 256 rows of 128 values, maximum and sum; eight numbers a block.
PMM_EXPORT long long pmm_tree_attention_scratch(int sms) { return static_cast<long long>(sms) * (2 * 2 * pmm::kTtRows * (128 + 2) + 8); }

PMM_EXPORT int pmm_tree_attention_tc(const void* q, long long ldq, const void* k, long long ldk, const void* v, long long ldv, const void* pool,
                                     int pages, const int* block_table, int max_blocks, const int* held, const int* cu, const int* positions,
                                     const void* mask, int words, const float* sink, void* out, float scale, int window, int window_step, int page_size,
                                     int n_seq, int T, int Hq, int Hkv, int Dh, int wide, float* scratch, int sms, int* status, cudaStream_t stream) {
  if (T <= 0 || n_seq <= 0) return 0;
  if (!tree_tc_supported(Hq, Hkv, Dh, page_size, pages, n_seq) || max_blocks <= 0 || !(scale > 0.f) || (window != 0 && !positions) ||
      (mask && words < 1) || !scratch || sms < 1 || !status)
    return PMM_ERR_BAD_ARGUMENT;
  for (const void* p : {q, k, v, pool, static_cast<const void*>(out), static_cast<const void*>(scratch)})
    if (reinterpret_cast<uintptr_t>(p) % 16) return PMM_ERR_BAD_ARGUMENT;
  const long long kv_dim = static_cast<long long>(Hkv) * Dh;
  if (T == 1) {  // (a matrix of one row has no stride of its own)
    ldq = static_cast<long long>(Hq) * Dh;
    ldk = ldv = kv_dim;
  }
  if (ldq % 8 || ldk % 8 || ldv % 8) return PMM_ERR_BAD_ARGUMENT;
  if (pmm::tree_attention_overlap(q, ldq, k, ldk, v, ldv, pool, pages, out, page_size, T, Hq, Hkv, Dh, 2)) return PMM_ERR_OVERLAP;
  pmm::EncodeTiledFn fn = pmm::encode_tiled_fn();
  if (!fn) return PMM_ERR_BAD_ARGUMENT;
  const int box = page_size % 64 == 0 ? 64 : page_size % 32 == 0 ? 32 : page_size % 16 == 0 ? 16 : 8;
  pmm::TreeMaps maps;
  bool ok = true;
  auto encode = [&](CUtensorMap* map, const void* base, long long n, long long ld, int box_rows) {
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(kv_dim), static_cast<cuuint64_t>(n)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld) * 2};
    const cuuint32_t boxes[2] = {pmm::kAtDhBlock, static_cast<cuuint32_t>(box_rows)};
    const cuuint32_t elem[2] = {1, 1};
    ok = ok && fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, boxes, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
  };
  encode(&maps.pool, pool, static_cast<long long>(pages) * 2 * page_size, kv_dim, box);
  encode(&maps.own_k, k, T, ldk, pmm::kAtBox);
  encode(&maps.own_v, v, T, ldv, pmm::kAtBox);
  if (!ok) return PMM_ERR_BAD_ARGUMENT;
  pmm::TreeTcArgs a{};
  a.q = static_cast<const pmm::bf16*>(q);
  a.ldq = ldq;
  a.v = static_cast<const pmm::bf16*>(v);
  a.ldv = ldv;
  a.pool = static_cast<const pmm::bf16*>(pool);
  a.block_table = block_table;
  a.max_blocks = max_blocks;
  a.pages = pages;
  a.held = held;
  a.cu = cu;
  a.positions = positions;
  a.mask = static_cast<const unsigned long long*>(mask);
  a.words = words;
  a.sink = sink;
  a.out = static_cast<pmm::bf16*>(out);
  a.shares = sms;
  a.rows = wide ? 2 * pmm::kTtRows : pmm::kTtRows;
  a.part_o = reinterpret_cast<float4*>(scratch);
  a.part_ml = reinterpret_cast<float2*>(scratch + static_cast<size_t>(a.shares) * 2 * a.rows * Dh);
  a.cuts = reinterpret_cast<int*>(scratch + static_cast<size_t>(a.shares) * 2 * a.rows * (Dh + 2));
  a.scale_log2 = scale * 1.4426950408889634f;
  a.window = window;
  a.window_step = window != 0 && window_step;
  a.page_size = page_size;
  a.box = box;
  a.n_seq = n_seq;
  a.T = T;
  a.Hq = Hq;
  a.Hkv = Hkv;
  a.status = status;
  if (Dh == 64) return wide ? pmm::launch_tree_tc<64, true>(maps, a, stream) : pmm::launch_tree_tc<64, false>(maps, a, stream);
  return wide ? pmm::launch_tree_tc<128, true>(maps, a, stream) : pmm::launch_tree_tc<128, false>(maps, a, stream);
}
