// Attention of drafted tokens over a paged cache on the fifth-generation tensor cores (the formulas of tree_attention.cu;
// bfloat16, head size 64 or 128, pages of a multiple of 8 positions).
//
// A unit of work is 64 or 128 rows (a row: a token and a query head of the group) of ONE request and ONE key/value head; its
// keys are tiles of 128, first the request's cached keys, then its own tokens of this step.  The number of tiles of all units
// is only known on the device (lengths are tensors, contexts are ragged), so every block adds it up and takes an equal share
// of the tiles, one behind the other (148 SMs stay busy to the end whatever the batch).  A unit that lies within one share is
// finished by its block; of a unit that shares cut, every block leaves (maximum, sum, unnormalised result) in scratch and a
// second launch merges them in the order of the keys, so results do not depend on which block came first.
// Within a block the roles and the walk over a tile are those of attention_tc.cu: warp 0 brings K and V tiles by TMA (cached
// keys in boxes that lie inside a page, the step's own from k and v) into a ring of three, warp 1 issues S = Q K^T and
// O += P V, a warp per 16 rows turns S into P with four threads per row.  The ring and the products run on across units: while
// a unit's result is written the next one's tiles travel, and its queries are put in place before.
// Of a tile's values only the 16 keys at a time that hold a valid one are multiplied; rows behind the last valid one (stale
// places of a page, other requests' tokens) are set to zero first, for 0 * NaN is NaN.  Where a tile's keys are not seen by
// all rows alike (the step's own tokens, a window's edge) values that are not finite are taken out of the product and added
// by hand to the rows that see them.
// Every mbarrier wait is bounded (status codes 41..45, see attention_tc.cu).  No cluster multicast.
#include "attention_tc.cuh"
#include <math_constants.h>

namespace pmm {

constexpr int kTtSeqs = 1024;  // requests whose lengths fit shared memory

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
template <int M>
__device__ __forceinline__ TreeSeq tree_seq(const TreeTcArgs& a, int t0, int t1, int held, int first) {
  TreeSeq s;
  s.t0 = t0;
  s.n_new = t1 - t0;
  s.held = held;
  s.first = first;
  const int G = a.Hq / a.Hkv;
  s.n_rt = (s.n_new * G + M - 1) / M;
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
template <int M, int THREADS>
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
      const TreeSeq q = tree_seq<M>(a, t0, t1, held, first);
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
template <int M>
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
  g.s = tree_seq<M>(a, p.cu[lo], p.cu[lo + 1], p.held[lo], p.first[lo]);
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

template <int DH, int M>
__global__ void __launch_bounds__(at_threads(M), DH == 64 ? 2 : 1)
    tree_attention_tc_kernel(const __grid_constant__ CUtensorMap map_kv, const __grid_constant__ CUtensorMap map_k,
                             const __grid_constant__ CUtensorMap map_v, const __grid_constant__ TreeTcArgs a) {
  constexpr int NSUB = DH / kAtDhBlock;
  constexpr int kThreads = at_threads(M);
  constexpr int kWarps = M / 16;
  constexpr int kQSub = at_q_sub(M);
  constexpr int kSlot = NSUB * kAtKvSub;
  constexpr unsigned kOff = at_o_offset(M);
  extern __shared__ unsigned char smem_raw[];
  __shared__ __align__(8) unsigned long long bar_q, bar_full[kAtRing], bar_empty[kAtRing], bar_s, bar_sfree, bar_p, bar_pv;
  __shared__ unsigned s_tmem_base;
  __shared__ int s_abort, s_red[32], s_bad[2];

  unsigned char* tiles = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* sQ = tiles;
  unsigned char* sRing = sQ + NSUB * kQSub;
  unsigned char* sP = sRing + kAtRing * kSlot;
  TreePlan plan;
  plan.pre = reinterpret_cast<int*>(sP + 2 * kQSub);
  plan.cu = plan.pre + a.n_seq + 1;
  plan.held = plan.cu + a.n_seq + 1;
  plan.first = plan.held + a.n_seq;

  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const int G = a.Hq / a.Hkv;
  pdl_launch_dependents();
  if (tid == 0) {
    mbar_init(&bar_q, kWarps);
#pragma unroll
    for (int i = 0; i < kAtRing; ++i) {
      mbar_init(&bar_full[i], 1);
      mbar_init(&bar_empty[i], 1);
    }
    mbar_init(&bar_s, 1);
    mbar_init(&bar_sfree, kWarps);
    mbar_init(&bar_p, kWarps);
    mbar_init(&bar_pv, 1);
    s_abort = 0;
    s_bad[0] = s_bad[1] = -1;
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    asm volatile("prefetch.tensormap [%0];\n" ::"l"(reinterpret_cast<unsigned long long>(&map_kv)) : "memory");
  }
  pdl_wait();
  tree_plan<M, kThreads>(a, plan, s_red);
  const int total = plan.pre[a.n_seq];
  const int shares = tree_shares(a, total);
  if (static_cast<int>(blockIdx.x) >= shares || total == 0) return;
  const int begin = tree_begin(blockIdx.x, total, shares), end = tree_begin(blockIdx.x + 1, total, shares);
  const int n_tiles = end - begin;  // (at least one)
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(&s_tmem_base)), "r"(at_tmem_cols(M)) : "memory");
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
      int row, boxes, hk;  // this lane's box: its row of the pool or of k and v; how many boxes; negative: the step's own tokens
    };
    auto request = [&](const Tile& t, bool is_v) {
      const int slot = item % kAtRing;
      if (item >= kAtRing && ok) {
        int got = 1;
        if (lane == 0) got = mbar_wait(&bar_empty[slot], (item / kAtRing - 1) & 1, abort_flag) ? 1 : 0;
        ok = __shfl_sync(0xffffffffu, got, 0) != 0;
        if (!ok && lane == 0) give_up(42);
      }
      if (!ok) return;
      const bool own = t.boxes < 0;
      const int boxes = own ? -t.boxes : t.boxes, rows = own ? kAtBox : a.box;
      if (lane == 0) mbar_expect_tx(&bar_full[slot], static_cast<unsigned>(boxes * rows * NSUB * 128));
      __syncwarp();
      const int b = lane / NSUB, d = lane % NSUB;
      const int row = __shfl_sync(0xffffffffu, t.row, b);
      if (b < boxes) {
        unsigned char* dst = sRing + slot * kSlot + d * kAtKvSub + b * rows * 128;
        const CUtensorMap* map = own ? (is_v ? &map_v : &map_k) : &map_kv;
        tma_load_2d(dst, map, t.hk * DH + d * kAtDhBlock, row + (is_v && !own ? page_size : 0), &bar_full[slot]);
      }
      ++item;
    };
    Tile prev{};
    for (int at = begin; at < end && ok;) {
      const TreeSeg g = tree_seg<M>(a, plan, at, end);
      const int* bt = a.block_table + static_cast<size_t>(g.seq) * a.max_blocks;
      int batch = g.j0 * per - 32, batch_row = 0;  // a lane's box of the 32 whose rows are at hand
      for (int j = g.j0; j < g.j1 && ok; ++j, ++at) {
        Tile t;
        const int valid = tree_valid(g.s, j);
        t.hk = g.hk;
        if (j < g.s.ctx_tiles) {
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
          t.boxes = (valid + a.box - 1) / a.box;
        } else {
          t.row = g.s.t0 + (j - g.s.ctx_tiles) * kAtKeys + lane * kAtBox;
          t.boxes = -((valid + kAtBox - 1) / kAtBox);
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
      for (int it = max(0, item - kAtRing); it < item; ++it)
        for (unsigned i = 0; i < kSpinLimit && !mbar_try_wait(&bar_full[it % kAtRing], (it / kAtRing) & 1); ++i) {
        }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA issuer (the whole warp walks, one lane issues)
    const int items = 2 * n_tiles;
    const unsigned lead = lane == 0 ? 1u : 0u;
    const unsigned long long q_desc = umma_desc(sQ), p_desc = umma_desc(sP), ring_desc = umma_desc(sRing);
    auto wait = [&](unsigned long long* bar, unsigned parity) {
      const bool got = mbar_wait(bar, parity, abort_flag);
      __syncwarp();  // (no lane may fall a phase behind)
      return got;
    };
    auto full = [&](int it) { return wait(&bar_full[it % kAtRing], (it / kAtRing) & 1); };
    auto issue_s = [&](int j) {  // S_j = Q K_j^T
      const int slot = at_k_item(j) % kAtRing;
      const unsigned long long k_desc = ring_desc + static_cast<unsigned>(slot * (kSlot >> 4));
#pragma unroll
      for (int k = 0; k < DH / 16; ++k)
        umma_f16_lead(tmem_base, q_desc + (k >> 2) * (kQSub >> 4) + 2 * (k & 3), k_desc + (k >> 2) * (kAtKvSub >> 4) + 2 * (k & 3),
                      at_idesc_s(M), k > 0 ? 1u : 0u, lead);
      umma_commit_lead(&bar_s, lead);
      if (at_k_item(j) + kAtRing < items) umma_commit_lead(&bar_empty[slot], lead);
    };
    int code = 0, segs = 0;
    TreeSeg g = tree_seg<M>(a, plan, begin, end);
    if (wait(&bar_q, 0) && full(0)) {
      asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
      issue_s(0);
    } else {
      code = 43;
    }
    for (int j = 0; j < n_tiles && code == 0; ++j) {
      const int own = begin + j - g.unit;  // this tile within its unit
      const int steps = (tree_valid(g.s, own) + 15) / 16;
      const bool fresh = own == g.j0;      // the first tile of a stretch: O begins anew
      if (own + 1 == g.j1) {               // the next tile is another unit's
        ++segs;
        if (j + 1 < n_tiles) g = tree_seg<M>(a, plan, begin + j + 1, end);
      }
      if (j + 1 < n_tiles) {
        // the softmax threads hold S_j in registers: the next S may overwrite it, and the tensor core works on it while they compute
        if (!full(at_k_item(j + 1)) || !wait(&bar_sfree, j & 1) || (begin + j + 1 == g.unit + g.j0 && !wait(&bar_q, segs & 1))) {
          code = 43;
          break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
        issue_s(j + 1);
      }
      const int v_item = at_v_item(j, n_tiles);
      if (!full(v_item) || !wait(&bar_p, j & 1)) {
        code = 44;
        break;
      }
      asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
      const int slot = v_item % kAtRing;
      const unsigned long long v_desc = ring_desc + static_cast<unsigned>(slot * (kSlot >> 4));
#pragma unroll
      for (int d = 0; d < NSUB; ++d)
#pragma unroll
        for (int k = 0; k < kAtKeys / 16; ++k)
          if (k < steps)
            umma_f16_lead(tmem_base + kOff + d * kAtDhBlock, p_desc + (k / 4) * (kQSub >> 4) + 2 * (k % 4),
                          v_desc + d * (kAtKvSub >> 4) + ((k * 16 * 128) >> 4), at_idesc_o(M), (!fresh || k > 0) ? 1u : 0u, lead);
      umma_commit_lead(&bar_pv, lead);
      if (v_item + kAtRing < items) umma_commit_lead(&bar_empty[slot], lead);
    }
    if (code != 0) give_up(code);
  } else {
    // ---------------------------------------------------------------- softmax and output (a warp per 16 rows)
    const int half = (warp - 2) >> 2;
    const int base_row = M == 64 ? (warp & 3) * 16 : (warp & 3) * 32 + half * 16;
    const unsigned lane_base = tmem_base + (static_cast<unsigned>((warp & 3) * 32 + half * 16) << 16);
    const int k4 = lane & 3;                              // this thread's columns: 4 i + k4
    const unsigned sel = (k4 & 1) ? 0x3276u : 0x5410u;    // see at_pair
    unsigned char* p_row = sP + ((k4 & 1) * 2 + (k4 >> 1)) * 4;
    const int row0 = base_row + (lane >> 2);
    const int soft_tid = tid - 64;                        // among the softmax threads
    bool alive = true;
    int gt = 0;                                           // tiles so far
    // the stretch's query rows -> shared memory, swizzled (rows beyond the unit are zero)
    auto queries = [&](const TreeSeg& g) {
      const int n_rows = min(M, g.s.n_new * G - g.rt * M);
      uint4 piece[DH / 16];
#pragma unroll
      for (int i = 0; i < DH / 16; ++i) {
        const int p = lane + 32 * i, rr = base_row + p / (DH / 8), c = p % (DH / 8);
        const int r = g.rt * M + rr, tk = r / G;
        piece[i] = rr < n_rows ? *reinterpret_cast<const uint4*>(a.q + (g.s.t0 + tk) * a.ldq + (g.hk * G + (r - tk * G)) * DH + c * 8)
                               : make_uint4(0u, 0u, 0u, 0u);
      }
#pragma unroll
      for (int i = 0; i < DH / 16; ++i) {
        const int p = lane + 32 * i, rr = base_row + p / (DH / 8), c = p % (DH / 8);
        *reinterpret_cast<uint4*>(sQ + (c >> 3) * kQSub + at_swizzled(rr, c & 7)) = piece[i];
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar_q);
    };
    TreeSeg g = tree_seg<M>(a, plan, begin, end);
    queries(g);
    for (int seg = 0, at = begin; at < end && alive; ++seg) {
      const int n_rows = min(M, g.s.n_new * G - g.rt * M);
      const bool idle = base_row >= n_rows;               // (the whole warp: none of its rows exists)
      int my_tok[2], my_lo[2];                            // of this thread's rows: token of the request, first cached key
      float m_run[2], l_run[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int row = row0 + 8 * r;
        my_tok[r] = row < n_rows ? (g.rt * M + row) / G : 0;
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
        const int last = (g.rt * M + n_rows - 1) / G;
        for (int tk = g.rt * M / G + lane; tk <= last; tk += 32) edge = max(edge, first_visible(a.positions[g.s.t0 + tk], a.window));
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
              w[0] >>= k4;
              w[1] >>= k4;
#pragma unroll
              for (int i = 0; i < kAtKeys / 4; ++i)
                if (!(w[i >> 4] >> (4 * (i & 15)) & 1ull)) v[2 * i + r] = __float_as_uint(-CUDART_INF_F);
            }
          } else if (valid < kAtKeys || base < max(my_lo[0], my_lo[1])) {
#pragma unroll
            for (int i = 0; i < kAtKeys / 4; ++i) {
              const int key = base + 4 * i + k4;
#pragma unroll
              for (int r = 0; r < 2; ++r)
                if (!(key >= my_lo[r] && key < g.s.held)) v[2 * i + r] = __float_as_uint(-CUDART_INF_F);
            }
          }
        }
        if (valid % 16 != 0 || mixed(g, j)) {
          // values that must not meet a probability of zero: rows behind the last valid one become zero; where rows see the
          // keys differently, so do values that are not finite
          const int item = at_v_item(gt, n_tiles), slot = item % kAtRing;
          ok = mbar_wait(&bar_full[slot], (item / kAtRing) & 1, abort_flag);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) {
            if (lane == 0) give_up(45);
            alive = false;
            break;
          }
          unsigned char* sV = sRing + slot * kSlot;
          const int from = mixed(g, j) ? 0 : valid * (DH / 8), to = (valid + 15) / 16 * 16 * (DH / 8);
          for (int p = from + soft_tid; p < to; p += kWarps * 32) {
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
          if (j > g.j0) {
            // P V_{j-1} must have finished: it read the P tile that is written below, and it wrote O
            ok = mbar_wait(&bar_pv, (gt - 1) & 1, abort_flag);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) {
              if (lane == 0) give_up(45);
              alive = false;
              break;
            }
            if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
              asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
#pragma unroll
              for (int c = 0; c < DH / 32; ++c) {
                unsigned ov[16];
                at_tmem_ld32(lane_base + kOff + c * 32, ov);
                asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
#pragma unroll
                for (int e = 0; e < 16; ++e) ov[e] = __float_as_uint(__uint_as_float(ov[e]) * alpha[e & 1]);
                at_tmem_st32(lane_base + kOff + c * 32, ov);
              }
              asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
            }
          }
          // P: four columns of both rows at a time, the exponentials of one group ahead of the packing of the one before
          sum[0] = sum[1] = 0.f;
          float p[2][4];
          auto exps = [&](int e0, float* dst) {
#pragma unroll
            for (int e = 0; e < 4; ++e) dst[e] = at_ex2(fmaf(__uint_as_float(v[4 * e0 + e]), a.scale_log2, -mu[e & 1]));
          };
          exps(0, p[0]);
#pragma unroll
          for (int e0 = 0; e0 < kAtKeys / 8; ++e0) {
            float* cur = p[e0 & 1];
            if (e0 + 1 < kAtKeys / 8) exps(e0 + 1, p[(e0 + 1) & 1]);
            unsigned char* dst = p_row + (e0 >> 3) * kQSub + at_swizzled(row0, e0 & 7);
            sum[0] += cur[0];
            sum[1] += cur[1];
            sum[0] += cur[2];
            sum[1] += cur[3];
            *reinterpret_cast<unsigned*>(dst) = at_pair(cur[0], cur[2], sel);
            *reinterpret_cast<unsigned*>(dst + 1024) = at_pair(cur[1], cur[3], sel);
          }
        } else if (j > g.j0) {
          // (a warp without rows keeps pace with the products: it must not be two phases ahead of any barrier)
          ok = mbar_wait(&bar_pv, (gt - 1) & 1, abort_flag);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) {
            if (lane == 0) give_up(45);
            alive = false;
            break;
          }
        }
        asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar_p);
      }
      if (!alive) break;
      if (!idle) take_sums();
      const TreeSeg now = g;
      if (at < end) {  // the next stretch's queries: the products of this one's have read theirs
        g = tree_seg<M>(a, plan, at, end);
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
          const float sk = a.sink[now.hk * G + (now.rt * M + row0 + 8 * r) % G] * 1.4426950408889634f;
          const float m_new = fmaxf(m_run[r], sk);
          corr[r] = exp2f(m_run[r] - m_new);
          l_run[r] = l_run[r] * corr[r] + exp2f(sk - m_new);
          m_run[r] = m_new;
        }
      }
      {
        bool ok = mbar_wait(&bar_pv, (gt - 1) & 1, abort_flag);
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
          at_tmem_ld(lane_base + kOff + c * 64, o);
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
          if (whole) {  // the rows go out in whole pieces, through this warp's rows of P's tiles
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              unsigned char* dst = p_row + c * kQSub + at_swizzled(row0, e);
#pragma unroll
              for (int r = 0; r < 2; ++r)
                *reinterpret_cast<unsigned*>(dst + 1024 * r) = at_pair(__uint_as_float(o[4 * e + r]) * inv[r], __uint_as_float(o[4 * e + 2 + r]) * inv[r], sel);
            }
          } else {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              if (!row_ok[r]) continue;
              float* dst = a.part_o + (slot * M + row0 + 8 * r) * DH + c * 64 + k4;
#pragma unroll
              for (int i = 0; i < 16; ++i) dst[4 * i] = __uint_as_float(o[2 * i + r]);
              if (c == 0 && k4 == 0) a.part_ml[slot * M + row0 + 8 * r] = make_float2(m_run[r], l_run[r]);
            }
          }
        }
        if (whole) {
          __syncwarp();
#pragma unroll
          for (int i = 0; i < DH / 16; ++i) {
            const int p = lane + 32 * i, rr = base_row + p / (DH / 8), c = p % (DH / 8);
            const int r = now.rt * M + rr, tk = r / G;
            if (rr < n_rows)
              *reinterpret_cast<uint4*>(a.out + (static_cast<size_t>(now.s.t0 + tk) * a.Hq + now.hk * G + (r - tk * G)) * DH + c * 8) =
                  *reinterpret_cast<const uint4*>(sP + (c >> 3) * kQSub + at_swizzled(rr, c & 7));
          }
          __syncwarp();
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
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem_base), "r"(at_tmem_cols(M)) : "memory");
  }
}

// Units that the shares cut: block (x, y) takes the unit that holds the first tile of share x + 1, where the share in front of it
// holds the unit's beginning, and the y-th piece of its rows.
//   M = max m_i;  o = sum_i o_i 2^(m_i - M) / sum_i l_i 2^(m_i - M)
constexpr int kTmThreads = 128;

template <int DH, int M>
__global__ void __launch_bounds__(kTmThreads) tree_merge_kernel(const __grid_constant__ TreeTcArgs a) {
  extern __shared__ int plan_mem[];
  __shared__ int s_red[32];
  pdl_launch_dependents();
  pdl_wait();
  TreePlan plan;
  plan.pre = plan_mem;
  plan.cu = plan.pre + a.n_seq + 1;
  plan.held = plan.cu + a.n_seq + 1;
  plan.first = plan.held + a.n_seq;
  tree_plan<M, kTmThreads>(a, plan, s_red);
  const int total = plan.pre[a.n_seq];
  if (total == 0) return;
  const int shares = tree_shares(a, total);
  const int share = blockIdx.x + 1;
  if (share >= shares) return;
  const int at = tree_begin(share, total, shares);
  const TreeSeg g = tree_seg<M>(a, plan, at, total);
  if (g.j0 == 0 || g.unit < tree_begin(share - 1, total, shares)) return;  // not cut here, or an earlier block's
  const int last = tree_block(g.unit + g.s.nt - 1, total, shares);
  const int G = a.Hq / a.Hkv, n_rows = min(M, g.s.n_new * G - g.rt * M);
  constexpr int C4 = DH / 4;
  constexpr int kBatch = 4;
  for (int i = blockIdx.y * kTmThreads + threadIdx.x; i < n_rows * C4; i += gridDim.y * kTmThreads) {
    const int r = i / C4, d = (i % C4) * 4;
    const int row = g.rt * M + r, tk = row / G, hq = g.hk * G + (row - tk * G);
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
        ml[u] = a.part_ml[slot * M + r];
        x[u] = *reinterpret_cast<const float4*>(a.part_o + (slot * M + r) * DH + d);
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

template <int DH, int M>
int launch_tree_tc(const CUtensorMap& kv, const CUtensorMap& k, const CUtensorMap& v, TreeTcArgs a, int sms, cudaStream_t stream) {
  const size_t smem = at_smem(DH, M) + tree_plan_bytes(a.n_seq);
  auto kern = tree_attention_tc_kernel<DH, M>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, 100);
  if (e != cudaSuccess) return static_cast<int>(e);
  launch_pdl(kern, dim3(a.shares), dim3(at_threads(M)), smem, stream, kv, k, v, a);
  const int st = launch_status();
  if (st != 0 || a.shares == 1) return st;
  launch_pdl(tree_merge_kernel<DH, M>, dim3(a.shares - 1, (M * DH / 4 + 2 * kTmThreads - 1) / (2 * kTmThreads)), dim3(kTmThreads),
             tree_plan_bytes(a.n_seq), stream, a);
  return launch_status();
}

}  // namespace pmm

// Whether pmm_tree_attention_tc takes this shape.
PMM_EXPORT int pmm_tree_attention_tc_supported(int Hq, int Hkv, int Dh, int page_size, long long pages, int n_seq) {
  if (Hkv <= 0 || Hq % Hkv) return 0;
  return ((Dh == 64 || Dh == 128) && page_size > 0 && page_size % 8 == 0 && pages > 0 && pages * 2 * page_size <= 0x7fffffffll && n_seq <= pmm::kTtSeqs)
             ? 1 : 0;
}

// Floats of scratch for `sms` multiprocessors: two parts a block of 128 rows of 128 values, maximum and sum, two blocks a multiprocessor
// with rows of 64 values.
PMM_EXPORT long long pmm_tree_attention_scratch(int sms) { return static_cast<long long>(sms) * 2 * 2 * 128 * (128 + 2); }

PMM_EXPORT int pmm_tree_attention_tc(const void* q, long long ldq, const void* k, long long ldk, const void* v, long long ldv, const void* pool,
                                     int pages, const int* block_table, int max_blocks, const int* held, const int* cu, const int* positions,
                                     const void* mask, int words, const float* sink, void* out, float scale, int window, int page_size, int n_seq,
                                     int T, int Hq, int Hkv, int Dh, int rows, float* scratch, int sms, int* status, cudaStream_t stream) {
  if (T <= 0 || n_seq <= 0) return 0;
  if (!pmm_tree_attention_tc_supported(Hq, Hkv, Dh, page_size, pages, n_seq) || max_blocks <= 0 || !(scale > 0.f) || (window != 0 && !positions) ||
      (mask && words < 1) || (rows != 64 && (rows != 128 || Dh != 128)) || !scratch || sms < 1 || !status)
    return PMM_ERR_BAD_ARGUMENT;
  for (const void* p : {q, k, v, pool, static_cast<const void*>(out), static_cast<const void*>(scratch)})
    if (reinterpret_cast<uintptr_t>(p) % 16) return PMM_ERR_BAD_ARGUMENT;
  if (ldq % 8 || ldk % 8 || ldv % 8) return PMM_ERR_BAD_ARGUMENT;
  pmm::EncodeTiledFn fn = pmm::encode_tiled_fn();
  if (!fn) return PMM_ERR_BAD_ARGUMENT;
  const int box = page_size % 64 == 0 ? 64 : page_size % 32 == 0 ? 32 : page_size % 16 == 0 ? 16 : 8;
  const long long kv_dim = static_cast<long long>(Hkv) * Dh;
  CUtensorMap maps[3];
  auto encode = [&](CUtensorMap* map, const void* base, long long n, long long ld, int box_rows) {
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(kv_dim), static_cast<cuuint64_t>(n)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld) * 2};
    const cuuint32_t boxes[2] = {pmm::kAtDhBlock, static_cast<cuuint32_t>(box_rows)};
    const cuuint32_t elem[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, boxes, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
  };
  // (a matrix of one row has no stride of its own)
  if (!encode(&maps[0], pool, static_cast<long long>(pages) * 2 * page_size, kv_dim, box) ||
      !encode(&maps[1], k, T, T > 1 ? ldk : kv_dim, pmm::kAtBox) || !encode(&maps[2], v, T, T > 1 ? ldv : kv_dim, pmm::kAtBox))
    return PMM_ERR_BAD_ARGUMENT;
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
  a.shares = sms * (Dh == 64 ? 2 : 1);
  a.part_o = scratch;
  a.part_ml = reinterpret_cast<float2*>(scratch + static_cast<size_t>(a.shares) * 2 * rows * Dh);
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
  if (Dh == 64) return pmm::launch_tree_tc<64, 64>(maps[0], maps[1], maps[2], a, sms, stream);
  return rows == 64 ? pmm::launch_tree_tc<128, 64>(maps[0], maps[1], maps[2], a, sms, stream)
                    : pmm::launch_tree_tc<128, 128>(maps[0], maps[1], maps[2], a, sms, stream);
}
