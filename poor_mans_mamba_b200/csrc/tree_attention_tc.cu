// Attention of drafted tokens over a paged cache on the fifth-generation tensor cores (the formulas of tree_attention.cu;
// bfloat16, head size 64 or 128, pages of a multiple of 16 positions).
//
// A unit of work is up to 128 rows (a row: a token and a query head of the group) of ONE request and ONE key/value head; its
// keys are tiles of 128, first the request's cached keys, then its own tokens of this step.  The number of tiles of all units
// is only known on the device (lengths are tensors, contexts are ragged), so every block adds it up and takes an equal share
// of the tiles, one behind the other (148 SMs stay busy to the end whatever the batch).  A unit that lies within one share is
// finished by its block; of a unit that shares cut, every block leaves (maximum, sum, unnormalised result) in scratch and a
// second launch merges them in the order of the keys, so results do not depend on which block came first.
// Within a block warp 0 brings K and V tiles by TMA (cached keys in boxes that lie inside a page, the step's own from k and
// v) into a ring, warp 1 issues S = Q K^T and O += P V, a warp per 16 rows turns S into P with four threads per row.  The ring
// and the products run on across units: while a unit's result is written the next one's tiles travel, and its queries are
// put in place before.
// Q and P are operands in tensor memory (Q, S, O and two tiles of P: 448 columns of 512): with both in shared memory a tile
// moves 64 KB in, 128 KB out to the products and 32 KB of P, 1,800 clocks at 128 bytes a clock, where the products take 1,026
// (eight of 128 x 128 x 16 each, 64 clocks; with half as many rows they take as long, so a unit has 128).  From tensor
// memory the products read K and V alone.  What thread k of a row's four holds of S are columns 4 i + k; as an operand, P has two
// neighbouring keys in a word.  So a K tile lies in shared memory with its even keys first and its odd keys behind them (two
// tensor maps of every other row): columns i and i + 16 of a thread are neighbouring keys, and no word changes threads.
// Of a tile's values only the 16 keys at a time that hold a valid one are multiplied; rows behind the last valid one (stale
// places of a page, other requests' tokens) are set to zero first, for 0 * NaN is NaN.  Where a tile's keys are not seen by
// all rows alike (the step's own tokens, a window's edge) values that are not finite are taken out of the product and added
// by hand to the rows that see them.
// Every mbarrier wait is bounded (status codes 41..45, see attention_tc.cu).  No cluster multicast.
#include "attention_tc.cuh"
#include <math_constants.h>

namespace pmm {

constexpr int kTtSeqs = 1024;  // requests whose lengths fit shared memory
constexpr int kTtRows = 128;   // rows of a unit
constexpr int kTtWarps = kTtRows / 16;
constexpr int kTtThreads = 64 + kTtWarps * 32;
// tensor memory: S, O, Q and two tiles of P (operands: two bfloat16 a column)
constexpr unsigned kTtO = 128, kTtQ = 256, kTtP = 320, kTtCols = 512;
__host__ __device__ constexpr int tree_ring(int dh) { return dh == 64 ? 11 : 6; }  // tiles in flight (16 or 32 KB each)
__host__ __device__ constexpr size_t tree_smem(int dh) { return static_cast<size_t>(tree_ring(dh)) * (dh / kAtDhBlock) * kAtKvSub + 1024 /*alignment*/; }

// S = Q K^T: both K-major; O += P V: V as it lies in the cache (MN-major), all DH columns at once.
constexpr unsigned kTtIdescS = at_idesc_s(kTtRows);
__host__ __device__ constexpr unsigned tree_idesc_o(int dh) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | (static_cast<unsigned>(dh >> 3) << 17) | (static_cast<unsigned>(kTtRows >> 4) << 24);
}
// A product whose A operand lies in tensor memory (row i in lane i, two neighbouring elements a column).
__device__ __forceinline__ void umma_ts_lead(unsigned tmem_d, unsigned tmem_a, unsigned long long b_desc, unsigned idesc, unsigned accumulate, unsigned lead) {
  asm volatile(
      "{\n\t.reg .pred p, l;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 l, %5, 0;\n\t"
      "@l tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n"
      :
      : "r"(tmem_d), "r"(tmem_a), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(lead)
      : "memory");
}
// The store that mirrors at_tmem_ld: 16 lanes of tensor memory x 64 columns.
__device__ __forceinline__ void tree_tmem_st(unsigned taddr, const unsigned* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x128b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};\n"
      :
      : "r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]),
        "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]),
        "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

// Tensor maps, two-dimensional with boxes of 64 columns: the pool's rows as they are (values), its even and its odd rows (keys), the
// step's values, the even and the odd rows of its keys.
struct TreeMaps {
  CUtensorMap pool_v, pool_k[2], own_v, own_k[2];
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
  float* part_o;        // [2 * blocks][M][DH]
  float2* part_ml;      // [2 * blocks][M]
  float scale_log2;
  int window, page_size, box, n_seq, T, Hq, Hkv, shares, min_tiles;
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
  s.n_rt = (s.n_new * G + kTtRows - 1) / kTtRows;
  s.ctx_tiles = held > first ? (held - first + kAtKeys - 1) / kAtKeys : 0;
  s.nt = s.ctx_tiles + (s.n_new + kAtKeys - 1) / kAtKeys;
  return s;
}

// The lengths of all requests in shared memory, and the running sum of their tiles.
struct TreePlan {
  int* pre;    // [n_seq + 1] tiles in front of a request
  int* cu;     // [n_seq + 1]
  int* held;   // [n_seq]
  int* first;  // [n_seq]
};
__host__ __device__ constexpr size_t tree_plan_bytes(int n_seq) { return (4 * static_cast<size_t>(n_seq) + 2) * sizeof(int); }

// Called by all THREADS threads of the block; red: shared memory for 32 ints.
template <int THREADS>
__device__ __forceinline__ void tree_plan(const TreeTcArgs& a, const TreePlan& p, int* red) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int total = 0;
  for (int base = 0; base < a.n_seq; base += THREADS) {
    const int s = base + tid;
    int tiles = 0;
    if (s < a.n_seq) {
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
      const TreeSeq q = tree_seq(a, t0, t1, held, first);
      tiles = q.nt * q.n_rt * a.Hkv;
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
}

// How many blocks share `total` tiles, the tile at which block b's share begins, and the block in whose share tile x lies.
__device__ __forceinline__ int tree_shares(const TreeTcArgs& a, int total) { return max(1, min(a.shares, total / a.min_tiles)); }
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
  int lo = 0, hi = a.n_seq - 1;  // the last request that begins at or before `at` (behind requests without tiles)
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (p.pre[mid] <= at)
      lo = mid;
    else
      hi = mid - 1;
  }
  TreeSeg g;
  g.seq = lo;
  g.s = tree_seq(a, p.cu[lo], p.cu[lo + 1], p.held[lo], p.first[lo]);
  const int off = at - p.pre[lo], u = off / g.s.nt;
  g.hk = u / g.s.n_rt;
  g.rt = u - g.hk * g.s.n_rt;
  g.unit = at - (off - u * g.s.nt);
  g.j0 = at - g.unit;
  g.j1 = min(g.s.nt, end - g.unit);
  return g;
}
// Valid keys of tile j.
__device__ __forceinline__ int tree_valid(const TreeSeq& s, int j) {
  return j < s.ctx_tiles ? min(kAtKeys, s.held - s.first - j * kAtKeys) : min(kAtKeys, s.n_new - (j - s.ctx_tiles) * kAtKeys);
}

template <int DH>
__global__ void __launch_bounds__(kTtThreads, 1) tree_attention_tc_kernel(const __grid_constant__ TreeMaps maps, const __grid_constant__ TreeTcArgs a) {
  constexpr int NSUB = DH / kAtDhBlock;
  constexpr int kRing = tree_ring(DH);
  constexpr int kSlot = NSUB * kAtKvSub;
  extern __shared__ unsigned char smem_raw[];
  __shared__ __align__(8) unsigned long long bar_q, bar_full[kRing], bar_empty[kRing], bar_s, bar_sfree, bar_p[2], bar_pv[2];
  __shared__ unsigned s_tmem_base;
  __shared__ int s_abort, s_red[32], s_bad[2];

  unsigned char* sRing = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  TreePlan plan;
  plan.pre = reinterpret_cast<int*>(sRing + kRing * kSlot);
  plan.cu = plan.pre + a.n_seq + 1;
  plan.held = plan.cu + a.n_seq + 1;
  plan.first = plan.held + a.n_seq;

  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const int G = a.Hq / a.Hkv;
  if (tid == 0) {
    mbar_init(&bar_q, kTtWarps);
#pragma unroll
    for (int i = 0; i < kRing; ++i) {
      mbar_init(&bar_full[i], 1);
      mbar_init(&bar_empty[i], 1);
    }
    mbar_init(&bar_s, 1);
    mbar_init(&bar_sfree, kTtWarps);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar_p[i], kTtWarps);
      mbar_init(&bar_pv[i], 1);
    }
    s_abort = 0;
    s_bad[0] = s_bad[1] = -1;
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    asm volatile("prefetch.tensormap [%0];\n" ::"l"(reinterpret_cast<unsigned long long>(&maps.pool_v)) : "memory");
  }
  pdl_wait();
  pdl_launch_dependents();  // (behind the wait: the merge reads the lengths ahead of its own)
  tree_plan<kTtThreads>(a, plan, s_red);
  const int total = plan.pre[a.n_seq];
  const int shares = tree_shares(a, total);
  if (static_cast<int>(blockIdx.x) >= shares || total == 0) return;
  const int begin = tree_begin(blockIdx.x, total, shares), end = tree_begin(blockIdx.x + 1, total, shares);
  const int n_tiles = end - begin;  // (at least one)
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(&s_tmem_base)), "r"(kTtCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
  const unsigned tmem_base = s_tmem_base;
  volatile int* abort_flag = &s_abort;
  auto give_up = [&](int code) {
    if (!*abort_flag) atomicExch(a.status, code);
    s_abort = 1;
  };

  if (warp == 0) {
    // ---------------------------------------------------------------- TMA producer (the whole warp walks, a lane a box)
    const int page_size = a.page_size;
    const int per = kAtKeys / a.box;  // boxes of a tile of cached keys
    int item = 0;
    bool ok = true;
    struct Tile {
      int row, valid, hk;  // row of the pool (of k and v) at which this lane's box begins, keys of the tile
      bool own;            // the step's own tokens
    };
    auto request = [&](const Tile& t, bool is_v) {
      const int slot = item % kRing;
      if (item >= kRing && ok) {
        int got = 1;
        if (lane == 0) got = mbar_wait(&bar_empty[slot], (item / kRing - 1) & 1, abort_flag) ? 1 : 0;
        ok = __shfl_sync(0xffffffffu, got, 0) != 0;
        if (!ok && lane == 0) give_up(42);
      }
      if (!ok) return;
      const int keys = t.own ? kAtBox : a.box;  // of a box
      const int boxes = (t.valid + keys - 1) / keys;
      if (lane == 0) mbar_expect_tx(&bar_full[slot], static_cast<unsigned>(boxes * keys * NSUB * 128));
      __syncwarp();
      // a lane a copy: box, sub-tile of 64 columns and, of keys, even or odd rows
      const int d = lane % NSUB, e = is_v ? 0 : lane / NSUB & 1, b = lane / (is_v ? NSUB : 2 * NSUB);
      const int row = __shfl_sync(0xffffffffu, t.row, b);
      if (b < boxes) {
        unsigned char* dst = sRing + slot * kSlot + d * kAtKvSub;
        const int col = t.hk * DH + d * kAtDhBlock;
        if (is_v)
          tma_load_2d(dst + b * keys * 128, t.own ? &maps.own_v : &maps.pool_v, col, row + (t.own ? 0 : page_size), &bar_full[slot]);
        else  // key 2 m + e of the tile to row 64 e + m
          tma_load_2d(dst + (64 * e + b * keys / 2) * 128, t.own ? &maps.own_k[(row + e) & 1] : &maps.pool_k[e], col, (row + (t.own ? e : 0)) >> 1,
                      &bar_full[slot]);
      }
      ++item;
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
      for (int it = max(0, item - kRing); it < item; ++it)
        for (unsigned i = 0; i < kSpinLimit && !mbar_try_wait(&bar_full[it % kRing], (it / kRing) & 1); ++i) {
        }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA issuer (the whole warp walks, one lane issues)
    // (what the products are issued with is known to be the same in the whole warp: it stays in uniform registers)
    auto uniform = [](auto x) { return __shfl_sync(0xffffffffu, x, 0); };
    const int n = uniform(n_tiles), items = 2 * n;
    const unsigned tmem = uniform(tmem_base);
    const unsigned lead = lane == 0 ? 1u : 0u;
    const unsigned long long ring_desc = umma_desc(sRing);
    // (of a V tile: 64 columns further lie one sub-tile further)
    const unsigned long long v_ring = (ring_desc & ~(0x3fffull << 16)) | (static_cast<unsigned long long>(kAtKvSub >> 4) << 16);
    auto wait = [&](unsigned long long* bar, unsigned parity) {
      const bool got = mbar_wait(bar, parity, abort_flag);
      __syncwarp();  // (no lane may fall a phase behind)
      return got;
    };
    auto full = [&](int it) { return wait(&bar_full[it % kRing], (it / kRing) & 1); };
    auto issue_s = [&](int j) {  // S_j = Q K_j^T
      const int slot = at_k_item(j) % kRing;
      const unsigned long long k_desc = ring_desc + static_cast<unsigned>(slot * (kSlot >> 4));
#pragma unroll
      for (int k = 0; k < DH / 16; ++k)
        umma_ts_lead(tmem, tmem + kTtQ + 8 * k, k_desc + (k >> 2) * (kAtKvSub >> 4) + 2 * (k & 3), kTtIdescS, k > 0 ? 1u : 0u, lead);
      umma_commit_lead(&bar_s, lead);
      if (at_k_item(j) + kRing < items) umma_commit_lead(&bar_empty[slot], lead);
    };
    int code = 0, segs = 0;
    TreeSeg g = tree_seg(a, plan, begin, end);
    if (wait(&bar_q, 0) && full(0)) {
      asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
      issue_s(0);
    } else {
      code = 43;
    }
    for (int j = 0; j < n && code == 0; ++j) {
      const int own = begin + j - g.unit;  // this tile within its unit
      const int steps = uniform((tree_valid(g.s, own) + 15) / 16);
      const unsigned more = uniform(own > g.j0 ? 1u : 0u);  // 0 in the first tile of a stretch: O begins anew
      if (own + 1 == g.j1) {               // the next tile is another unit's
        ++segs;
        if (j + 1 < n) g = tree_seg(a, plan, begin + j + 1, end);
      }
      if (j + 1 < n) {
        // the softmax threads hold S_j in registers: the next S may overwrite it, and the tensor core works on it while they compute
        if (!full(at_k_item(j + 1)) || !wait(&bar_sfree, j & 1) || (begin + j + 1 == g.unit + g.j0 && !wait(&bar_q, segs & 1))) {
          code = 43;
          break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
        issue_s(j + 1);
      }
      const int v_item = at_v_item(j, n);
      if (!full(v_item) || !wait(&bar_p[j & 1], (j >> 1) & 1)) {
        code = 44;
        break;
      }
      asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
      const int slot = v_item % kRing;
      const unsigned long long v_desc = v_ring + static_cast<unsigned>(slot * (kSlot >> 4));
      const unsigned p_tmem = tmem + kTtP + 64 * (j & 1);
      auto product = [&](int k) {  // 16 keys: 16 rows of 128 bytes of every sub-tile
        umma_ts_lead(tmem + kTtO, p_tmem + 8 * k, v_desc + ((k * 16 * 128) >> 4), tree_idesc_o(DH), k > 0 ? 1u : more, lead);
      };
      if (steps == kAtKeys / 16) {
#pragma unroll
        for (int k = 0; k < kAtKeys / 16; ++k) product(k);
      } else {
        for (int k = 0; k < steps; ++k) product(k);
      }
      umma_commit_lead(&bar_pv[j & 1], lead);
      if (v_item + kRing < items) umma_commit_lead(&bar_empty[slot], lead);
    }
    if (code != 0) give_up(code);
  } else {
    // ---------------------------------------------------------------- softmax and output (a warp per 16 rows)
    // groups of 16 rows go round the four quarters of tensor memory (and of the multiprocessor): few rows, too, use all of it
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    const int base_row = (half * 4 + quarter) * 16;
    const unsigned lane_base = tmem_base + (static_cast<unsigned>(quarter * 32 + half * 16) << 16);
    const int k4 = lane & 3;                              // this thread's columns: 4 i + k4
    const int row0 = base_row + (lane >> 2);
    const int soft_tid = tid - 64;                        // among the softmax threads
    bool alive = true;
    int gt = 0;                                           // tiles so far
    auto product_done = [&](int i) { return mbar_wait(&bar_pv[i & 1], (i >> 1) & 1, abort_flag); };  // O += P V of tile i
    // the stretch's query rows -> tensor memory (rows beyond the unit are zero)
    auto queries = [&](const TreeSeg& g) {
      const int n_rows = min(kTtRows, g.s.n_new * G - g.rt * kTtRows);
      unsigned w[DH / 4];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int row = row0 + 8 * r, gr = g.rt * kTtRows + row, tk = gr / G;
        const bool there = row < n_rows;
        const unsigned* src = reinterpret_cast<const unsigned*>(a.q + (g.s.t0 + (there ? tk : 0)) * a.ldq + (g.hk * G + (there ? gr - tk * G : 0)) * DH) + k4;
#pragma unroll
        for (int i = 0; i < DH / 8; ++i) w[2 * i + r] = there ? src[4 * i] : 0u;
      }
#pragma unroll
      for (int c = 0; c < DH / 64; ++c) at_tmem_st32(lane_base + kTtQ + 32 * c, w + 16 * c);
      asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
      asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar_q);
    };
    TreeSeg g = tree_seg(a, plan, begin, end);
    queries(g);
    for (int seg = 0, at = begin; at < end && alive; ++seg) {
      const int n_rows = min(kTtRows, g.s.n_new * G - g.rt * kTtRows);
      const bool idle = base_row >= n_rows;               // (the whole warp: none of its rows exists)
      int my_tok[2], my_lo[2];                            // of this thread's rows: token of the request, first cached key
      float m_run[2], l_run[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int row = row0 + 8 * r;
        my_tok[r] = row < n_rows ? (g.rt * kTtRows + row) / G : 0;
        my_lo[r] = a.window != 0 ? first_visible(a.positions[g.s.t0 + my_tok[r]], a.window) : 0;
        m_run[r] = -CUDART_INF_F;
        l_run[r] = 0.f;
      }
      float sum[2] = {0.f, 0.f}, alpha[2] = {1.f, 1.f};
      auto take_sums = [&]() {
        float t0 = sum[0] + __shfl_xor_sync(0xffffffffu, sum[0], 1), t1 = sum[1] + __shfl_xor_sync(0xffffffffu, sum[1], 1);
        t0 += __shfl_xor_sync(0xffffffffu, t0, 2);
        t1 += __shfl_xor_sync(0xffffffffu, t1, 2);
        l_run[0] = l_run[0] * alpha[0] + t0;
        l_run[1] = l_run[1] * alpha[1] + t1;
      };
      // the bits of a row's visible keys among the 128 of tile j of the step's own tokens
      auto own_bits = [&](int r, int j, unsigned long long (&w)[2]) {
        const int k0 = (j - g.s.ctx_tiles) * kAtKeys, valid = tree_valid(g.s, j);
        const int upto = a.mask ? valid : min(valid, my_tok[r] + 1 - k0);  // without masks: up to the token itself
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int n = upto - 64 * h;
          w[h] = n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1ull;
          if (a.mask) {
            const int at_word = k0 / 64 + h;
            w[h] &= at_word < a.words ? a.mask[static_cast<size_t>(g.s.t0 + my_tok[r]) * a.words + at_word] : 0ull;
          }
        }
      };
      int edge = 0;                                       // behind it every row of the unit sees all cached keys
      if (a.window != 0) {
        const int last = (g.rt * kTtRows + n_rows - 1) / G;
        for (int tk = g.rt * kTtRows / G + lane; tk <= last; tk += 32) edge = max(edge, first_visible(a.positions[g.s.t0 + tk], a.window));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) edge = max(edge, __shfl_xor_sync(0xffffffffu, edge, o));
      }
      // whether the rows may see tile j's keys differently: the step's own tokens, and in front of the windows' last edge
      auto mixed = [&](const TreeSeg& of, int j) { return j >= of.s.ctx_tiles || of.s.first + j * kAtKeys < edge; };
      for (int j = g.j0; j < g.j1; ++j, ++gt, ++at) {
        const bool own = j >= g.s.ctx_tiles;
        const int base = g.s.first + j * kAtKeys;         // (cached keys)
        const int valid = tree_valid(g.s, j);
        bool ok = mbar_wait(&bar_s, gt & 1, abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) {
          if (lane == 0) give_up(45);
          alive = false;
          break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
        unsigned v[kAtKeys / 2];
        if (!idle) {
          at_tmem_ld(lane_base, v);
          at_tmem_ld(lane_base + 64, v + 32);
          if (j > g.j0) take_sums();  // (of the tile before, while these travel)
          asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
        }
        asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar_sfree);
        if (!idle) {
          if (own) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              unsigned long long w[2];
              own_bits(r, j, w);
              w[0] >>= 2 * k4;
              w[1] >>= 2 * k4;
#pragma unroll
              for (int i = 0; i < kAtKeys / 4; ++i)  // keys 8 (i % 16) + 2 k4 + i / 16
                if (!(w[(i & 15) >> 3] >> (8 * (i & 7) + (i >> 4)) & 1ull)) v[2 * i + r] = __float_as_uint(-CUDART_INF_F);
            }
          } else if (valid < kAtKeys || base < max(my_lo[0], my_lo[1])) {
#pragma unroll
            for (int i = 0; i < kAtKeys / 4; ++i) {
              const int key = base + 8 * (i & 15) + 2 * k4 + (i >> 4);
#pragma unroll
              for (int r = 0; r < 2; ++r)
                if (!(key >= my_lo[r] && key < g.s.held)) v[2 * i + r] = __float_as_uint(-CUDART_INF_F);
            }
          }
        }
        if (valid % 16 != 0 || mixed(g, j)) {
          // values that must not meet a probability of zero: rows behind the last valid one become zero; where rows see the
          // keys differently, so do values that are not finite
          const int item = at_v_item(gt, n_tiles), slot = item % kRing;
          ok = mbar_wait(&bar_full[slot], (item / kRing) & 1, abort_flag);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) {
            if (lane == 0) give_up(45);
            alive = false;
            break;
          }
          unsigned char* sV = sRing + slot * kSlot;
          const int from = mixed(g, j) ? 0 : valid * (DH / 8), to = (valid + 15) / 16 * 16 * (DH / 8);
          for (int p = from + soft_tid; p < to; p += kTtWarps * 32) {
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
        if (!idle) {
          float mx[2][2];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            mx[r][0] = fmaxf(__uint_as_float(v[r]), __uint_as_float(v[2 + r]));
            mx[r][1] = fmaxf(__uint_as_float(v[4 + r]), __uint_as_float(v[6 + r]));
          }
#pragma unroll
          for (int i = 4; i < kAtKeys / 4; i += 4)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              mx[r][0] = at_max3(mx[r][0], __uint_as_float(v[2 * i + r]), __uint_as_float(v[2 * i + 2 + r]));
              mx[r][1] = at_max3(mx[r][1], __uint_as_float(v[2 * i + 4 + r]), __uint_as_float(v[2 * i + 6 + r]));
            }
          mx[0][0] = fmaxf(mx[0][0], mx[0][1]);
          mx[1][0] = fmaxf(mx[1][0], mx[1][1]);
#pragma unroll
          for (int o = 1; o <= 2; ++o) {
            const float o0 = __shfl_xor_sync(0xffffffffu, mx[0][0], o), o1 = __shfl_xor_sync(0xffffffffu, mx[1][0], o);
            mx[0][0] = fmaxf(mx[0][0], o0);
            mx[1][0] = fmaxf(mx[1][0], o1);
          }
          float mu[2];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float m = mx[r][0] * a.scale_log2;  // scale > 0
            // raise the maximum in use only when the row's maximum has run ahead of it by more than kAtLazy
            const bool raise = (m > m_run[r] + kAtLazy || m_run[r] == -CUDART_INF_F) && m != -CUDART_INF_F;
            alpha[r] = raise ? at_ex2(m_run[r] - m) : 1.f;
            m_run[r] = raise ? m : m_run[r];
            mu[r] = (m_run[r] == -CUDART_INF_F) ? 0.f : m_run[r];
          }
          const bool rescale = j > g.j0 && __any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f);
          if (gt >= 2 || rescale) {
            // the product of two tiles ago must have finished: it read the P tile that is written below; the one before
            // this tile's, too, where its sums are to be scaled (rare)
            ok = gt < 2 || product_done(gt - 2);
            if (rescale) ok = ok && product_done(gt - 1);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) {
              if (lane == 0) give_up(45);
              alive = false;
              break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
            if (rescale) {
#pragma unroll
              for (int c = 0; c < DH / 32; ++c) {
                unsigned ov[16];
                at_tmem_ld32(lane_base + kTtO + c * 32, ov);
                asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
#pragma unroll
                for (int e = 0; e < 16; ++e) ov[e] = __float_as_uint(__uint_as_float(ov[e]) * alpha[e & 1]);
                at_tmem_st32(lane_base + kTtO + c * 32, ov);
              }
              asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
            }
          }
          // P, two neighbouring keys a word
          sum[0] = sum[1] = 0.f;
#pragma unroll
          for (int i = 0; i < 16; ++i)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const float p0 = at_ex2(fmaf(__uint_as_float(v[2 * i + r]), a.scale_log2, -mu[r]));  // masked: ex2(-inf) = 0
              const float p1 = at_ex2(fmaf(__uint_as_float(v[2 * (i + 16) + r]), a.scale_log2, -mu[r]));
              sum[r] += p0;
              sum[r] += p1;
              v[2 * i + r] = at_pack(p0, p1);
            }
          tree_tmem_st(lane_base + kTtP + 64 * (gt & 1), v);
          asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
        } else if (gt >= 2) {
          // (a warp without rows keeps pace with the products: it must not be two phases ahead of any barrier)
          ok = product_done(gt - 2);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) {
            if (lane == 0) give_up(45);
            alive = false;
            break;
          }
        }
        asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar_p[gt & 1]);
      }
      if (!alive) break;
      if (!idle) take_sums();
      const TreeSeg now = g;
      if (at < end) {  // the next stretch's queries: the products of this one's have read theirs
        g = tree_seg(a, plan, at, end);
        queries(g);
      }

      // ---- this stretch's result: O from tensor memory once the last product has finished
      const bool whole = now.j0 == 0 && now.j1 == now.s.nt;
      const bool row_ok[2] = {row0 < n_rows, row0 + 8 < n_rows};
      float corr[2] = {1.f, 1.f};
      if (a.sink != nullptr && whole) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          if (!row_ok[r]) continue;
          // a score without key or value that counts once; maxima are kept in units of log 2
          const float sk = a.sink[now.hk * G + (now.rt * kTtRows + row0 + 8 * r) % G] * 1.4426950408889634f;
          const float m_new = fmaxf(m_run[r], sk);
          corr[r] = exp2f(m_run[r] - m_new);
          l_run[r] = l_run[r] * corr[r] + exp2f(sk - m_new);
          m_run[r] = m_new;
        }
      }
      {
        bool ok = product_done(gt - 1);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) {
          if (lane == 0) give_up(45);
          alive = false;
          break;
        }
      }
      asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
      const bool repair = reinterpret_cast<volatile int*>(s_bad)[seg & 1] == seg;
      if (!idle) {
        const size_t slot = 2 * static_cast<size_t>(blockIdx.x) + (now.j0 > 0 ? 0 : 1);
        float inv[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) inv[r] = whole ? (l_run[r] == 0.f ? 0.f : corr[r] / l_run[r]) : 1.f;  // (NaN stays NaN)
#pragma unroll
        for (int c = 0; c < NSUB; ++c) {
          unsigned o[32];
          at_tmem_ld(lane_base + kTtO + c * 64, o);
          asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
          if (repair) {
            // values that are not finite, to the rows that see their keys
            for (int j = now.j0; j < now.j1; ++j) {
              const bool own = j >= now.s.ctx_tiles;
              if (!mixed(now, j)) continue;
              const int valid = tree_valid(now.s, j);
              for (int k = 0; k < valid; ++k) {
                const bf16* vr;
                const int key = now.s.first + j * kAtKeys + k, node = (j - now.s.ctx_tiles) * kAtKeys + k;
                if (own) {
                  vr = a.v + (now.s.t0 + node) * a.ldv + now.hk * DH;
                } else {
                  const int page = min(max(a.block_table[static_cast<size_t>(now.seq) * a.max_blocks + key / a.page_size], 0), a.pages - 1);
                  vr = a.pool + ((static_cast<long long>(page) * 2 + 1) * a.page_size + key % a.page_size) * a.Hkv * DH + now.hk * DH;
                }
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                  bool see;
                  if (own)
                    see = a.mask ? node < 64 * a.words && (a.mask[static_cast<size_t>(now.s.t0 + my_tok[r]) * a.words + (node >> 6)] >> (node & 63) & 1ull)
                                 : node <= my_tok[r];
                  else
                    see = key >= my_lo[r];
                  if (!see) continue;
#pragma unroll
                  for (int i = 0; i < 16; ++i) {
                    const float x = __bfloat162float(vr[c * 64 + 4 * i + k4]);
                    if (!(fabsf(x) < CUDART_INF_F)) o[2 * i + r] = __float_as_uint(__uint_as_float(o[2 * i + r]) + x);
                  }
                }
              }
            }
          }
          if (whole) {
            const unsigned sel = (k4 & 1) ? 0x3276u : 0x5410u;  // see at_pair
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const int gr = now.rt * kTtRows + row0 + 8 * r, tk = gr / G;
              unsigned* dst = reinterpret_cast<unsigned*>(a.out + (static_cast<size_t>(now.s.t0 + tk) * a.Hq + now.hk * G + (gr - tk * G)) * DH + c * 64) +
                              (k4 & 1) * 2 + (k4 >> 1);
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const unsigned word = at_pair(__uint_as_float(o[4 * e + r]) * inv[r], __uint_as_float(o[4 * e + 2 + r]) * inv[r], sel);
                if (row_ok[r]) dst[4 * e] = word;
              }
            }
          } else {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              if (!row_ok[r]) continue;
              float* dst = a.part_o + (slot * kTtRows + row0 + 8 * r) * DH + c * 64 + k4;
#pragma unroll
              for (int i = 0; i < 16; ++i) dst[4 * i] = __uint_as_float(o[2 * i + r]);
              if (c == 0 && k4 == 0) a.part_ml[slot * kTtRows + row0 + 8 * r] = make_float2(m_run[r], l_run[r]);
            }
          }
        }
      }
      // (the next stretch's first product into O comes behind this warp's arrival for its probabilities)
      asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
    }
  }

  asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
  __syncthreads();
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem_base), "r"(kTtCols) : "memory");
  }
}

// Units that the shares cut: block (x, y) takes the unit that holds the first tile of share x + 1, where the share in front of it
// holds the unit's beginning, and the y-th piece of its rows.
//   M = max m_i;  o = sum_i o_i 2^(m_i - M) / sum_i l_i 2^(m_i - M)
constexpr int kTmThreads = 128;

template <int DH>
__global__ void __launch_bounds__(kTmThreads) tree_merge_kernel(const __grid_constant__ TreeTcArgs a) {
  extern __shared__ int plan_mem[];
  __shared__ int s_red[32];
  pdl_launch_dependents();
  TreePlan plan;
  plan.pre = plan_mem;
  plan.cu = plan.pre + a.n_seq + 1;
  plan.held = plan.cu + a.n_seq + 1;
  plan.first = plan.held + a.n_seq;
  tree_plan<kTmThreads>(a, plan, s_red);  // (lengths and tables were there before the launch in front of this one passed its wait)
  pdl_wait();                                // (every block waits: the next launch takes this one's end for that of both)
  const int total = plan.pre[a.n_seq];
  if (total == 0) return;
  const int shares = tree_shares(a, total);
  const int share = blockIdx.x + 1;
  if (share >= shares) return;
  const int at = tree_begin(share, total, shares);
  const TreeSeg g = tree_seg(a, plan, at, total);
  if (g.j0 == 0 || g.unit < tree_begin(share - 1, total, shares)) return;  // not cut here, or an earlier block's
  const int last = tree_block(g.unit + g.s.nt - 1, total, shares);
  const int G = a.Hq / a.Hkv, n_rows = min(kTtRows, g.s.n_new * G - g.rt * kTtRows);
  constexpr int C4 = DH / 4;
  constexpr int kBatch = 4;
  for (int i = blockIdx.y * kTmThreads + threadIdx.x; i < n_rows * C4; i += gridDim.y * kTmThreads) {
    const int r = i / C4, d = (i % C4) * 4;
    const int row = g.rt * kTtRows + r, tk = row / G, hq = g.hk * G + (row - tk * G);
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
        ml[u] = a.part_ml[slot * kTtRows + r];
        x[u] = *reinterpret_cast<const float4*>(a.part_o + (slot * kTtRows + r) * DH + d);
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
    stf4(a.out + (static_cast<size_t>(g.s.t0 + tk) * a.Hq + hq) * DH + d, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
  }
}

template <int DH>
int launch_tree_tc(const TreeMaps& maps, const TreeTcArgs& a, cudaStream_t stream) {
  const size_t smem = tree_smem(DH) + tree_plan_bytes(a.n_seq);
  auto kern = tree_attention_tc_kernel<DH>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, 100);
  if (e != cudaSuccess) return static_cast<int>(e);
  launch_pdl(kern, dim3(a.shares), dim3(kTtThreads), smem, stream, maps, a);
  const int st = launch_status();
  if (st != 0 || a.shares == 1) return st;
  launch_pdl(tree_merge_kernel<DH>, dim3(a.shares - 1, kTtRows * DH / 4 / (2 * kTmThreads)), dim3(kTmThreads), tree_plan_bytes(a.n_seq), stream, a);
  return launch_status();
}

}  // namespace pmm

// Whether pmm_tree_attention_tc takes this shape.
PMM_EXPORT int pmm_tree_attention_tc_supported(int Hq, int Hkv, int Dh, int page_size, long long pages, int n_seq) {
  if (Hkv <= 0 || Hq % Hkv) return 0;
  return ((Dh == 64 || Dh == 128) && page_size > 0 && page_size % 16 == 0 && pages > 0 && pages * 2 * page_size <= 0x7fffffffll && n_seq <= pmm::kTtSeqs)
             ? 1 : 0;
}

// Floats of scratch for `sms` multiprocessors: two parts a block of 128 rows of 128 values, maximum and sum.
PMM_EXPORT long long pmm_tree_attention_scratch(int sms) { return static_cast<long long>(sms) * 2 * pmm::kTtRows * (128 + 2); }

PMM_EXPORT int pmm_tree_attention_tc(const void* q, long long ldq, const void* k, long long ldk, const void* v, long long ldv, const void* pool,
                                     int pages, const int* block_table, int max_blocks, const int* held, const int* cu, const int* positions,
                                     const void* mask, int words, const float* sink, void* out, float scale, int window, int page_size, int n_seq,
                                     int T, int Hq, int Hkv, int Dh, float* scratch, int sms, int* status, cudaStream_t stream) {
  if (T <= 0 || n_seq <= 0) return 0;
  if (!pmm_tree_attention_tc_supported(Hq, Hkv, Dh, page_size, pages, n_seq) || max_blocks <= 0 || !(scale > 0.f) || (window != 0 && !positions) ||
      (mask && words < 1) || !scratch || sms < 1 || !status)
    return PMM_ERR_BAD_ARGUMENT;
  for (const void* p : {q, k, v, pool, static_cast<const void*>(out), static_cast<const void*>(scratch)})
    if (reinterpret_cast<uintptr_t>(p) % 16) return PMM_ERR_BAD_ARGUMENT;
  if (ldq % 8 || ldk % 8 || ldv % 8) return PMM_ERR_BAD_ARGUMENT;
  pmm::EncodeTiledFn fn = pmm::encode_tiled_fn();
  if (!fn) return PMM_ERR_BAD_ARGUMENT;
  const int box = page_size % 64 == 0 ? 64 : page_size % 32 == 0 ? 32 : 16;
  const long long kv_dim = static_cast<long long>(Hkv) * Dh, pool_rows = static_cast<long long>(pages) * 2 * page_size;
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
  const pmm::bf16 *pool_b = static_cast<const pmm::bf16*>(pool), *k_b = static_cast<const pmm::bf16*>(k);
  if (T == 1) ldk = ldv = kv_dim;  // (a matrix of one row has no stride of its own)
  encode(&maps.pool_v, pool, pool_rows, kv_dim, box);
  encode(&maps.own_v, v, T, ldv, pmm::kAtBox);
  for (int e = 0; e < 2; ++e) {
    encode(&maps.pool_k[e], pool_b + e * kv_dim, pool_rows / 2, 2 * kv_dim, box / 2);
    const int odd = T > 1 ? e : 0;  // (of a single row there are no odd ones, and none is asked for)
    encode(&maps.own_k[e], k_b + odd * ldk, (T + 1 - odd) / 2, 2 * ldk, pmm::kAtBox / 2);
  }
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
  a.part_o = scratch;
  a.part_ml = reinterpret_cast<float2*>(scratch + static_cast<size_t>(a.shares) * 2 * pmm::kTtRows * Dh);
  a.scale_log2 = scale * 1.4426950408889634f;
  a.window = window;
  a.page_size = page_size;
  a.box = box;
  a.n_seq = n_seq;
  a.T = T;
  a.Hq = Hq;
  a.Hkv = Hkv;
  a.min_tiles = 2;
  a.status = status;
  return Dh == 64 ? pmm::launch_tree_tc<64>(maps, a, stream) : pmm::launch_tree_tc<128>(maps, a, stream);
}
