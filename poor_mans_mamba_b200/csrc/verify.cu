// Which drafted tokens the target model keeps, and the token behind them, from its logits and given random numbers.
//
// Row t of the logits is what the target says behind token t of the step; token 0 of a request is its root, the others are
// drafted.  With p = softmax(logits / T) and one uniform u per token:
//   drafts from a distribution (a chain, draft_logits given, q = softmax(draft_logits / T)): token i behind its parent is kept
//     when u_i q(x_i) < p(x_i) and all before it are; behind the first that is not the next token is drawn from
//     max(p - q, 0), behind the last from p, each with the root's uniform;
//   fixed proposals (a chain or a tree): t is drawn from p with the node's uniform, the walk goes to the first child that
//     holds t, and where none does t is the next token.
// Both leave a token distributed as p.  "Drawn with u": the first index whose running sum of weights passes u times their
// total.  T <= 0: the largest logit, the first on ties, in the place of every draw.
// A NaN logit counts as -inf; +inf shares the weight among its like; a row without a finite or +inf logit draws token 0 and
// keeps no draft.  Where max(p - q, 0) has no weight left (it has some in exact arithmetic), p is drawn from.
//
// The answers are whole numbers behind comparisons of sums over some 10^5 weights: with weights rounded to 32 bits a draw in a
// hundred would come out differently from the formula, so what decides is in 64 bits (vf_exp2).  The 64-bit units do not keep
// pace with memory (32 clocks a weight and warp against 23 for the bytes), so not every row goes through them:
// First launch: a warp per (row, 1,024 entries) reads its entries once and leaves their maximum and the sum of
// exp((l - maximum) / T); for drafts with a distribution in 32 bits (the sums are off by less than 2^-17 of themselves), for
// fixed proposals, each node of which draws, in 64.
// Second launch: a cluster of up to 16 blocks per request.  With a draft's distribution, u q(x) < p(x) is decided from the first
// launch's sums where the sides are 2^-14 apart or more, else (hardly ever) from exact sums of the two rows; then the row
// that the next token is drawn from, and the draft's behind it, go once through the cluster's warps.  A draw is one block's work:
// it finds the piece of 1,024 by the pieces' sums and the entry in it, four entries a thread; a tree's nodes draw side by side.
#include "common.cuh"
#include <math_constants.h>

namespace pmm {

constexpr int kVfThreads = 256;
constexpr int kVfWarps = kVfThreads / 32;
constexpr int kVfEach = 32;
constexpr int kVfChunk = 32 * kVfEach;
constexpr int kVfCluster = 16;      // blocks of a cluster at most
constexpr int kVfChunksMax = 2048;  // sums of a row's pieces in shared memory
constexpr int kVfStep = 4;          // entries of a row that a lane takes at a time in the second launch
constexpr int kVfNear = 4;          // places that a lane remembers
constexpr int kVfNodes = 64;        // nodes of a chain whose rows' sums are kept

struct __align__(16) VfChunk {
  double sum;   // of exp((l - top) / T)
  float top;
  int at;       // the first index that holds top (only where T <= 0)
};

struct VerifyArgs {
  const float* logits;
  long long ld;
  const float* draft;       // or nullptr: fixed proposals
  long long ld_draft;
  const int* tokens;
  const int* parents;       // or nullptr: chains
  const int* cu;
  int n;
  const float* uniforms;
  const float* temperature; // [n] or nullptr: all greedy
  int V, n_rows, chunks;
  VfChunk* stats;           // [n_rows, chunks], then the same of the draft
  int* drawn;               // [n_rows]
  int* tokens_out;
  int* path;
  int width;
  int* count;
  int cluster;              // blocks that share a request
};

// 2^(y/32) for y in (-32000, 0], to 3e-15 of itself: 2^(k/32) from a table, k = round(y), times the exponential series of the rest,
// |y - k| ln 2 / 32 <= 0.0109, up to its fifth power (the scheme of Tang, Table-driven implementation of the exponential
// function, 1989).  y = 0 gives 1 exactly.
__device__ __forceinline__ double vf_exp2(double y, const double* table) {
  constexpr double kRound = 6755399441055744.0;  // 1.5 * 2^52: adding it leaves the nearest integer in the low bits
  constexpr double kLn = 0.69314718055994530942 / 32.0;
  const double t = y + kRound;
  const int k = __double2loint(t);
  const double r = y - (t - kRound);
  double p = kLn * kLn * kLn * kLn * kLn / 120.0;
  p = fma(p, r, kLn * kLn * kLn * kLn / 24.0);
  p = fma(p, r, kLn * kLn * kLn / 6.0);
  p = fma(p, r, kLn * kLn / 2.0);
  p = fma(p, r, kLn);
  p = fma(p, r, 1.0);
  const double power = table[k & 31];  // 2^(k % 32 / 32), less k % 32 in the place to which k is added
  return p * __hiloint2double(__double2hiint(power) + (k << 15), __double2loint(power));
}
__constant__ double kVfPowers[32] = {  // 2^(k/32)
    1.0, 1.0218971486541166, 1.0442737824274138, 1.0671404006768237,
    1.0905077326652577, 1.1143867425958924, 1.1387886347566916, 1.1637248587775775,
    1.189207115002721, 1.215247359980469, 1.241857812073484, 1.2690509571917332,
    1.2968395546510096, 1.3252366431597413, 1.3542555469368927, 1.383909881963832,
    1.4142135623730951, 1.4451808069770467, 1.4768261459394993, 1.5091644275934228,
    1.5422108254079407, 1.5759808451078865, 1.6104903319492543, 1.645755478153965,
    1.681792830507429, 1.718619298122478, 1.7562521603732995, 1.7947090750031072,
    1.8340080864093424, 1.8741676341103, 1.9152065613971474, 1.9571441241754002};
__device__ __forceinline__ void vf_table(double* table) {
  const int j = threadIdx.x;
  if (j < 32) table[j] = __hiloint2double(__double2hiint(kVfPowers[j]) - (j << 15), __double2loint(kVfPowers[j]));
}
// 32 log2(e) / T (temperatures outside 1e-36..1e36 count as the nearer of the two: no product below leaves its type)
__device__ __forceinline__ double vf_scale(float temp) { return 32.0 * 1.4426950408889634074 / fmin(fmax(static_cast<double>(temp), 1e-36), 1e36); }

__device__ __forceinline__ float vf_clean(float l) { return l == l ? l : -CUDART_INF_F; }

// exp((l - top) / T) as the formulas above want it at infinities; top is at least l.  (No branches: several of them run side by
// side, a chain of dependent 64-bit operations each.)
__device__ __forceinline__ double vf_weight(float l, float top, double c, const double* table) {
  // (beyond 2^-1000 of the largest a weight counts for nothing; a difference of infinities is no number and does not count either)
  const bool live = (l - top) * static_cast<float>(c) > -32000.f;
  const double w = vf_exp2((static_cast<double>(live ? l : 0.f) - static_cast<double>(live ? top : 0.f)) * c, table);
  return live ? w : top == CUDART_INF_F && l == top ? 1.0 : 0.0;
}

// 2^x to 2^-22 of itself, 0 below 2^-126 (what is smaller than that beside the largest weight, 1, counts for nothing).
__device__ __forceinline__ float vf_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}

// The request that row r belongs to: how many end at or before it.  Called by a whole warp.
__device__ __forceinline__ int vf_request(const int* cu, int n, int r) {
  int s = 0;
  for (int b = 0; b < n; b += 128) {  // four loads in flight
    int ends[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) ends[u] = cu[min(b + 32 * u + static_cast<int>(threadIdx.x & 31), n - 1) + 1];
    int c = 0;
#pragma unroll
    for (int u = 0; u < 4; ++u) c += __popc(__ballot_sync(0xffffffffu, b + 32 * u + static_cast<int>(threadIdx.x & 31) < n && ends[u] <= r));
    s += c;
    if (c < 128) break;
  }
  return s;
}

__device__ __forceinline__ double vf_sum(double x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}
// The larger of (top, at) over a warp, the lower place on ties.
__device__ __forceinline__ void vf_top(float& top, int& at) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float ot = __shfl_xor_sync(0xffffffffu, top, o);
    const int oa = __shfl_xor_sync(0xffffffffu, at, o);
    if (ot > top || (ot == top && oa < at)) {
      top = ot;
      at = oa;
    }
  }
}

// Whether all of a lane's N entries are numbers whose weights against `top` count.
template <int N>
__device__ __forceinline__ bool vf_counts(const float (&v)[N], float top, float scale) {
  float low = CUDART_INF_F, nan = 0.f;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    low = fminf(low, v[k]);
    nan = fmaf(v[k], 0.f, nan);  // NaN where an entry is NaN or infinite
  }
  return nan == 0.f && (low - top) * scale > -32000.f;
}

// EXACT: sums in 64 bits.
template <bool EXACT>
__global__ void __launch_bounds__(kVfThreads, 4) verify_stats_kernel(const VerifyArgs a) {
  __shared__ double s_table[32];
  pdl_launch_dependents();
  if (EXACT) {
    vf_table(s_table);
    __syncthreads();
  }
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const unsigned w = blockIdx.x * kVfWarps + (threadIdx.x >> 5);
  const int r = static_cast<int>(w / a.chunks), c = static_cast<int>(w % a.chunks);
  const bool of_draft = blockIdx.y == 1;
  if (r >= a.n_rows) return;
  const int base = c * kVfChunk + lane;
  const float* row = (of_draft ? a.draft + r * a.ld_draft : a.logits + r * a.ld) + base;
  float v[kVfEach];
  auto load = [&]() {
    if (c * kVfChunk + kVfChunk <= a.V) {
#pragma unroll
      for (int k = 0; k < kVfEach; ++k) v[k] = row[k * 32];
    } else {
#pragma unroll
      for (int k = 0; k < kVfEach; ++k) v[k] = base + k * 32 < a.V ? row[k * 32] : -CUDART_INF_F;
    }
  };
  if (!of_draft) load();  // (beside the request's search; not every row of the draft is wanted)
  const int s = vf_request(a.cu, a.n, r);
  if (s >= a.n) return;   // (behind the last request)
  const float temp = a.temperature ? a.temperature[s] : 0.f;
  const bool greedy = !(temp > 0.f);
  if (of_draft) {
    if (greedy || r == a.cu[s + 1] - 1) return;  // (nothing was drafted behind a chain's last token)
    load();
  }
  float top = -CUDART_INF_F;
  int at = base;
  double sum = 0.0;
  if (greedy) {
#pragma unroll
    for (int k = 0; k < kVfEach; ++k)
      if (v[k] > top) {  // (never true of NaN)
        top = v[k];
        at = base + k * 32;
      }
    vf_top(top, at);
  } else {
#pragma unroll
    for (int k = 0; k < kVfEach; ++k) top = fmaxf(top, v[k]);  // (NaN gives way)
    top = warp_max(top);
    const double scale = vf_scale(temp);
    if (top == CUDART_INF_F) {  // the infinite ones share the weight
#pragma unroll
      for (int k = 0; k < kVfEach; ++k) sum += v[k] == top ? 1.0 : 0.0;
    } else if (top > -CUDART_INF_F) {
      if (EXACT) {
        // What counts for nothing, NaN and -inf among it, is held at an exponent of -31900 / 32: a weight of 2^-997 leaves a sum of 1 and
        // more as it is.  The exponent is held, not the logit: beside a large maximum or a small temperature no float says "31900 less".
        // (It is not above 0, so of two numbers the lower one has the larger upper half.)
        const unsigned least = static_cast<unsigned>(__double2hiint(-31900.0));
        double part[2] = {0.0, 0.0};
#pragma unroll
        for (int k = 0; k < kVfEach; ++k) {
          const double y = (static_cast<double>(fmaxf(v[k], -CUDART_INF_F)) - static_cast<double>(top)) * scale;
          part[k & 1] += vf_exp2(__hiloint2double(static_cast<int>(min(static_cast<unsigned>(__double2hiint(y)), least)), __double2loint(y)), s_table);
        }
        sum = part[0] + part[1];
      } else {
        const float c2 = static_cast<float>(scale * 0.03125);
        float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < kVfEach; ++k) {
          const float x = (v[k] - top) * c2;
          part[k & 3] += fmaxf(vf_ex2(x), 0.f);  // (NaN gives way)
        }
        sum = (static_cast<double>(part[0]) + part[1]) + (static_cast<double>(part[2]) + part[3]);
      }
    }
    sum = vf_sum(sum);
  }
  if (lane == 0) a.stats[(static_cast<size_t>(of_draft ? a.n_rows : 0) + r) * a.chunks + c] = VfChunk{sum, top, at};
}

// A row's maximum (and its first place, of a greedy row), and the sum of exp((l - maximum) / T) over the row, by one warp.
struct VfRow {
  float top;
  int at;
  double sum;
};
__device__ __noinline__ VfRow vf_row(const VfChunk* st, int chunks, double scale, bool greedy, const double* table) {
  const int lane = threadIdx.x & 31;
  VfRow r{-CUDART_INF_F, 0, 0.0};
  for (int b = lane; b < chunks; b += 128) {  // four loads in flight
    VfChunk x[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) x[u] = st[min(b + 32 * u, chunks - 1)];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (x[u].top > r.top) {
        r.top = x[u].top;
        r.at = x[u].at;
      }
  }
  vf_top(r.top, r.at);
  if (greedy) return r;
  for (int b = lane; b < chunks; b += 128) {
    VfChunk x[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) x[u] = st[min(b + 32 * u, chunks - 1)];
#pragma unroll
    for (int u = 0; u < 4; ++u) r.sum += b + 32 * u < chunks ? x[u].sum * vf_weight(x[u].top, r.top, scale, table) : 0.0;
  }
  r.sum = vf_sum(r.sum);
  return r;
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}

struct VfShared {
  double table[32], scan[kVfWarps], left;
  int pick, last;
};

// The whole block: sum of x.
__device__ __forceinline__ double vf_block_sum(double x, VfShared& sh) {
  x = vf_sum(x);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh.scan[threadIdx.x >> 5] = x;
  __syncthreads();
  x = 0.0;
#pragma unroll
  for (int w = 0; w < kVfWarps; ++w) x += sh.scan[w];
  return x;
}
// The whole block: the first thread at which the running sum of x passes `target` (the last with any weight where rounding leaves
// none); `target` becomes what is left of it there.
__device__ __noinline__ int vf_block_find(double x, double& target, VfShared& sh) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  double run = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double up = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += up;
  }
  __syncthreads();
  if (lane == 31) sh.scan[warp] = run;
  if (tid == 0) {
    sh.pick = 0x7fffffff;
    sh.last = 0;
  }
  __syncthreads();
  double before = 0.0;
#pragma unroll
  for (int w = 0; w < kVfWarps; ++w)
    if (w < warp) before += sh.scan[w];
  const unsigned hit = __ballot_sync(0xffffffffu, x > 0.0 && before + run > target), any = __ballot_sync(0xffffffffu, x > 0.0);
  if (lane == 0) {
    if (hit) atomicMin(&sh.pick, warp * 32 + __ffs(hit) - 1);
    if (any) atomicMax(&sh.last, warp * 32 + 31 - __clz(any));
  }
  __syncthreads();
  const int pick = sh.pick != 0x7fffffff ? sh.pick : sh.last;
  if (tid == pick) sh.left = target - (before + run - x);
  __syncthreads();
  target = sh.left;
  return pick;
}
// The whole block: the first of n values part(i) (of n entries at most 256 * `each`) whose running sum passes `target`.
template <typename P>
__device__ __forceinline__ int vf_block_place(int n, double& target, VfShared& sh, P part) {
  const int each = (n + kVfThreads - 1) / kVfThreads, first = static_cast<int>(threadIdx.x) * each;
  double own = 0.0;
  for (int i = first; i < min(n, first + each); ++i) own += part(i);
  const int who = vf_block_find(own, target, sh);
  if (each == 1) return who;
  double run = 0.0, left = target;
  int at = who * each;
  for (int i = who * each; i < min(n, who * each + each); ++i) {  // (every thread walks them)
    const double x = part(i);
    if (x > 0.0) {
      at = i;
      left = target - run;
      if (run + x > target) break;
    }
    run += x;
  }
  target = left;
  return at;
}
// The whole block: the entry of piece c whose running sum of weight(i) passes `target`.
template <typename W>
__device__ __forceinline__ int vf_block_entry(int c, int V, double target, VfShared& sh, W weight) {
  constexpr int kFour = kVfChunk / kVfThreads;
  const int first = c * kVfChunk + static_cast<int>(threadIdx.x) * kFour;
  double x[kFour], own = 0.0;
#pragma unroll
  for (int k = 0; k < kFour; ++k) x[k] = first + k < V ? weight(first + k) : 0.0;
#pragma unroll
  for (int k = 0; k < kFour; ++k) own += x[k];
  const int who = vf_block_find(own, target, sh);
  if (static_cast<int>(threadIdx.x) == who) {
    double run = 0.0;
    int at = 0;
    bool found = false;
#pragma unroll
    for (int k = 0; k < kFour; ++k) {
      if (x[k] > 0.0 && !found) {
        at = k;
        found = run + x[k] > target;
      }
      run += x[k];
    }
    sh.pick = first + at;
  }
  __syncthreads();
  return sh.pick;
}

__global__ void __launch_bounds__(kVfThreads, 2) verify_walk_kernel(const VerifyArgs a) {
  extern __shared__ double s_part[];  // [4][chunks]: a piece's weight in p and in q, and the same of the entries with more in p than in q
  __shared__ VfShared sh;
  __shared__ VfRow s_row[2][kVfNodes], s_one;
  __shared__ int s_kept, s_ok[kVfNodes];
  vf_table(sh.table);
  __syncthreads();
  pdl_wait();
  const int cluster = a.cluster, s = blockIdx.x / cluster, rank = blockIdx.x % cluster, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int t0 = max(a.cu[s], 0), t1 = min(max(a.cu[s + 1], 0), a.n_rows);  // (no bound leads out of the rows)
  const int nodes = t1 - t0;
  const float temp = a.temperature ? a.temperature[s] : 0.f;
  const bool greedy = !(temp > 0.f);
  const double scale = greedy ? 0.0 : vf_scale(temp);
  int* out = a.tokens_out + static_cast<size_t>(s) * a.width;
  int* path = a.path + static_cast<size_t>(s) * a.width;
  if (nodes <= 0) {  // (the same for the whole cluster)
    if (rank == 0) {
      for (int j = tid; j < a.width; j += kVfThreads) out[j] = path[j] = -1;
      if (tid == 0) a.count[s] = 0;
      pdl_arrived();
    }
    return;
  }
  auto stats = [&](int r, bool of_draft) { return a.stats + (static_cast<size_t>(of_draft ? a.n_rows : 0) + r) * a.chunks; };
  // a draw from p of row r with u, by the whole block (-1: no token has any weight)
  auto draw = [&](int r, float u) {
    const VfChunk* st = stats(r, false);
    __syncthreads();
    if (warp == 0) {
      const VfRow got = vf_row(st, a.chunks, scale, greedy, sh.table);
      if (lane == 0) s_one = got;
    }
    __syncthreads();
    const VfRow one = s_one;
    if (one.top == -CUDART_INF_F) return -1;
    if (greedy) return one.at;
    double target = static_cast<double>(u) * one.sum;
    const int c = vf_block_place(a.chunks, target, sh, [&](int i) { return st[i].sum * vf_weight(st[i].top, one.top, scale, sh.table); });
    const float* row = a.logits + r * a.ld;
    return vf_block_entry(c, a.V, target, sh, [&](int i) { return vf_weight(vf_clean(row[i]), one.top, scale, sh.table); });
  };

  if (a.draft == nullptr) {
    // ---- fixed proposals: every node's draw, a block each; then the walk
    for (int i = rank; i < nodes; i += cluster) {
      const int got = draw(t0 + i, a.uniforms[t0 + i]);
      if (tid == 0) a.drawn[t0 + i] = got;
    }
    cluster_sync();
    if (rank != 0 || warp != 0) return;
    int now = 0, kept = 0;
    if (lane == 0) path[0] = 0;
    while (true) {
      const int want = __ldcg(a.drawn + t0 + now);
      int child = -1;
      if (want >= 0 && kept + 1 < a.width)
        for (int b = now + 1; b < nodes && child < 0; b += 32) {
          const int i = b + lane;
          bool is = false;
          if (i < nodes) {
            const int up = a.parents ? a.parents[t0 + i] : i - 1;
            is = up == now && a.tokens[t0 + i] == want;
          }
          const unsigned any = __ballot_sync(0xffffffffu, is);
          if (any) child = b + __ffs(any) - 1;
        }
      if (lane == 0) out[kept] = max(want, 0);
      if (child < 0) break;
      ++kept;
      if (lane == 0) path[kept] = child;
      now = child;
    }
    for (int j = kept + 1 + lane; j < a.width; j += 32) out[j] = path[j] = -1;
    if (lane == 0) a.count[s] = kept + 1;
    __threadfence();  // (as pdl_arrived: all that is left of the block is this warp)
    return;
  }

  // ---- a chain from a draft's distribution: which tokens are kept (every block of the cluster finds out for itself)
  // Row r of the target (and the draft's, `both`) once through all warps of the cluster: the pieces' weights in s_part of every block,
  // and the weights of the entries with more in p than in q in s_part of the block that took the piece.  The sums at hand tell which
  // those are but for the entries where p and q are within 2^-15 of one another: a lane remembers their places (`settle`).
  int near[kVfNear], n_near = 0;
  auto send = [&](int which, int c, double x) {  // to block lane % cluster
    unsigned dst;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n"
                 : "=r"(dst)
                 : "r"(static_cast<unsigned>(__cvta_generic_to_shared(s_part + which * a.chunks + c))), "r"(lane % cluster));
    asm volatile("st.shared::cluster.f64 [%0], %1;\n" ::"r"(dst), "d"(x) : "memory");
  };
  auto pass = [&](int r, const VfRow of_p, const VfRow of_q, bool both) {
    const float* row = a.logits + r * a.ld;
    const float* row_q = a.draft + r * a.ld_draft;
    const float scale_f = static_cast<float>(scale);
    const double inv = of_p.sum > 0.0 ? 1.0 / of_p.sum : 0.0, inv_q = of_q.sum > 0.0 ? 1.0 / of_q.sum : 0.0;
    n_near = 0;
    cluster_sync();  // (every block of the cluster is there, and done with what it held)
    for (int c = rank + cluster * warp; c < a.chunks; c += cluster * kVfWarps) {
      double sum_p = 0.0, sum_q = 0.0, more_p = 0.0, more_q = 0.0;
      const int base = c * kVfChunk + lane;
      // what an entry adds; whether p and q are too near to tell which is more there
      auto add = [&](double p, double q) {
        sum_p += p;
        sum_q += q;
        const double in_p = p * inv, more = fma(-q, inv_q, in_p);
        // |more| < 2^-15 in_p, by the halves that hold the exponents
        const bool tied = (__double2hiint(more) & 0x7fffffff) < __double2hiint(in_p) - (15 << 20);
        const bool take = !tied && __double2hiint(more) > 0;
        more_p += take ? p : 0.0;
        more_q += take ? q : 0.0;
        return tied;
      };
      auto remember = [&](int i) {
#pragma unroll
        for (int u = kVfNear - 1; u > 0; --u) near[u] = near[u - 1];
        near[0] = i;
        ++n_near;
      };
      auto slow = [&](int first, int n) {
#pragma unroll 1
        for (int i = first; i < min(a.V, first + n * 32); i += 32)
          if (add(vf_weight(vf_clean(row[i]), of_p.top, scale, sh.table), both ? vf_weight(vf_clean(row_q[i]), of_q.top, scale, sh.table) : 0.0)) remember(i);
      };
      if (c * kVfChunk + kVfChunk > a.V) {
        slow(base, kVfEach);
      } else {
        const float *at = row + base, *at_q = row_q + base;
        const double top_p = of_p.top, top_q = of_q.top;
        float v[kVfStep], v_q[kVfStep], w[kVfStep], w_q[kVfStep];  // some entries of both rows, and the next ones on their way
        auto fetch = [&](int k0, float (&x)[kVfStep], float (&y)[kVfStep]) {
#pragma unroll
          for (int k = 0; k < kVfStep; ++k) x[k] = at[(k0 + k) * 32];
          if (both) {
#pragma unroll
            for (int k = 0; k < kVfStep; ++k) y[k] = at_q[(k0 + k) * 32];
          }
        };
        auto take = [&](int i0, const float (&x)[kVfStep], const float (&y)[kVfStep]) {
          const bool fine = vf_counts<kVfStep>(x, of_p.top, scale_f) && (!both || vf_counts<kVfStep>(y, of_q.top, scale_f));
          if (!__all_sync(0xffffffffu, fine)) {
            slow(i0, kVfStep);
          } else if (both) {
            double p[kVfStep], q[kVfStep];
#pragma unroll
            for (int k = 0; k < kVfStep; ++k) {
              p[k] = vf_exp2((static_cast<double>(x[k]) - top_p) * scale, sh.table);
              q[k] = vf_exp2((static_cast<double>(y[k]) - top_q) * scale, sh.table);
            }
            unsigned tied = 0u;
#pragma unroll
            for (int k = 0; k < kVfStep; ++k) tied |= add(p[k], q[k]) ? 1u << k : 0u;
            if (tied) {
#pragma unroll
              for (int k = 0; k < kVfStep; ++k)
                if (tied >> k & 1u) remember(i0 + k * 32);
            }
          } else {
#pragma unroll
            for (int k = 0; k < kVfStep; ++k) {
              const double p = vf_exp2((static_cast<double>(x[k]) - top_p) * scale, sh.table);
              (k & 1 ? sum_q : sum_p) += p;  // (two chains; one sum in the end)
            }
          }
        };
        fetch(0, v, v_q);
#pragma unroll 1
        for (int k0 = 0; k0 < kVfEach; k0 += 2 * kVfStep, at += 2 * kVfStep * 32, at_q += 2 * kVfStep * 32) {
          fetch(kVfStep, w, w_q);
          take(base + k0 * 32, v, v_q);
          if (k0 + 2 * kVfStep < kVfEach) fetch(2 * kVfStep, v, v_q);
          take(base + (k0 + kVfStep) * 32, w, w_q);
        }
      }
      if (!both) {
        sum_p += sum_q;
        sum_q = 0.0;
      }
      sum_p = vf_sum(sum_p);
      if (both) {
        sum_q = vf_sum(sum_q);
        more_p = vf_sum(more_p);
        more_q = vf_sum(more_q);
      }
      if (lane < 2 * cluster) send(lane / cluster, c, lane / cluster == 0 ? sum_p : sum_q);
      if (lane == 0) {
        s_part[2 * a.chunks + c] = more_p;
        s_part[3 * a.chunks + c] = more_q;
      }
    }
    cluster_sync();
  };
  // The entries that were too near to tell, with the exact sums behind inv and inv_q; then the last two of s_part are in every block.
  auto settle = [&](int r, const VfRow of_p, const VfRow of_q, double inv, double inv_q) {
    const float* row = a.logits + r * a.ld;
    const float* row_q = a.draft + r * a.ld_draft;
    const bool lost = __any_sync(0xffffffffu, n_near > kVfNear);  // (more places than a lane remembers: the pieces once more)
    for (int c = rank + cluster * warp; c < a.chunks; c += cluster * kVfWarps) {
      double more_p = 0.0, more_q = 0.0;
      auto add = [&](int i) {
        const double p = vf_weight(vf_clean(row[i]), of_p.top, scale, sh.table), q = vf_weight(vf_clean(row_q[i]), of_q.top, scale, sh.table);
        if (p * inv > q * inv_q) {
          more_p += p;
          more_q += q;
        }
      };
      if (lost) {
#pragma unroll 1
        for (int i = c * kVfChunk + lane; i < min(a.V, c * kVfChunk + kVfChunk); i += 32) add(i);
      } else {
#pragma unroll
        for (int u = 0; u < kVfNear; ++u)
          if (u < n_near && near[u] / kVfChunk == c) add(near[u]);
      }
      more_p = vf_sum(more_p);
      more_q = vf_sum(more_q);
      if (!lost) {
        more_p += s_part[2 * a.chunks + c];
        more_q += s_part[3 * a.chunks + c];
      }
      __syncwarp();
      if (lane < 2 * cluster) send(2 + lane / cluster, c, lane / cluster == 0 ? more_p : more_q);
    }
    cluster_sync();
  };
  auto total = [&](int which) {
    double x = 0.0;
    for (int c = tid; c < a.chunks; c += kVfThreads) x += s_part[which * a.chunks + c];
    return vf_block_sum(x, sh);
  };
  const int drafted = min(nodes, a.width) - 1;
  int kept = 0;
  for (int first = 1; first <= drafted && kept == first - 1; first += kVfNodes) {  // (kVfNodes at a time, while all before are kept)
    const int n = min(kVfNodes, drafted - first + 1);
    __syncthreads();
    if (tid == 0) s_kept = first - 1 + n;
    // a warp a row: the target's rows and the draft's
    for (int j = warp; j < 2 * n; j += kVfWarps) {
      const int i = first + (j >> 1);
      if ((j & 1) && greedy) continue;
      const VfRow got = vf_row(stats(t0 + i - 1, j & 1), a.chunks, scale, greedy, sh.table);
      if (lane == 0) s_row[j & 1][i - first] = got;
    }
    __syncthreads();
    if (tid < n) {
      const int i = first + tid, r = t0 + i - 1, x = a.tokens[t0 + i];
      const VfRow of_p = s_row[0][tid];
      int ok = 0;
      if (greedy) {
        ok = of_p.at == x && of_p.top > -CUDART_INF_F;
      } else if (x >= 0 && x < a.V) {
        const VfRow of_q = s_row[1][tid];
        const double p = vf_weight(vf_clean(a.logits[r * a.ld + x]), of_p.top, scale, sh.table);
        const double q = vf_weight(vf_clean(a.draft[r * a.ld_draft + x]), of_q.top, scale, sh.table);
        // (a draft without weight anywhere proposes nothing that could be kept)
        if (of_p.sum > 0.0 && of_q.sum > 0.0) {
          const double left = static_cast<double>(a.uniforms[t0 + i]) * q * of_p.sum, right = p * of_q.sum;
          ok = left < right;
          if (fabs(left - right) <= 0x1p-14 * right) ok = 2;
        }
      }
      s_ok[tid] = ok;
      if (ok != 1) atomicMin(&s_kept, i - 1);
    }
    __syncthreads();
    kept = s_kept;
    while (kept < first - 1 + n && s_ok[kept + 1 - first] == 2) {  // too near to tell: by exact sums (the same for the whole cluster)
      const int j = kept + 1 - first, r = t0 + kept, x = a.tokens[t0 + kept + 1];
      pass(r, s_row[0][j], s_row[1][j], true);
      const double p = vf_weight(vf_clean(a.logits[r * a.ld + x]), s_row[0][j].top, scale, sh.table);
      const double q = vf_weight(vf_clean(a.draft[r * a.ld_draft + x]), s_row[1][j].top, scale, sh.table);
      if (!(static_cast<double>(a.uniforms[t0 + kept + 1]) * q * total(0) < p * total(1))) break;
      do ++kept;
      while (kept < first - 1 + n && s_ok[kept + 1 - first] == 1);
    }
    if (kept < first - 1 + n) break;
  }
  const int r = t0 + kept;
  int got = -1;
  if (greedy) {
    if (rank != 0) return;
    if (warp == 0) {
      const VfRow one = vf_row(stats(r, false), a.chunks, scale, true, sh.table);
      if (lane == 0) s_one = one;
    }
    __syncthreads();
    got = s_one.at;
  } else {
    const bool rest = kept < drafted;  // a draft was refused: what p has more than q
    VfRow of_p, of_q{};
    if (rest) {
      of_p = s_row[0][kept % kVfNodes];  // (the refused token's place among the last ones looked at)
      of_q = s_row[1][kept % kVfNodes];
    } else {
      __syncthreads();
      if (warp == 0) {
        const VfRow one = vf_row(stats(r, false), a.chunks, scale, false, sh.table);
        if (lane == 0) s_one = one;
      }
      __syncthreads();
      of_p = s_one;
    }
    pass(r, of_p, of_q, rest);
    const double sum = total(0);
    double inv = 0.0, inv_q = 0.0;
    if (rest) {
      const double sum_q = total(1);
      inv = sum > 0.0 ? 1.0 / sum : 0.0;
      inv_q = sum_q > 0.0 ? 1.0 / sum_q : 0.0;
      settle(r, of_p, of_q, inv, inv_q);
    }
    if (rank != 0) return;
    const float* row = a.logits + r * a.ld;
    const float* row_q = a.draft + r * a.ld_draft;
    const double u = static_cast<double>(a.uniforms[t0]);
    if (rest) {
      auto piece = [&](int c) { return fmax(s_part[2 * a.chunks + c] * inv - s_part[3 * a.chunks + c] * inv_q, 0.0); };
      double whole = 0.0;
      for (int c = tid; c < a.chunks; c += kVfThreads) whole += piece(c);
      whole = vf_block_sum(whole, sh);
      if (whole > 0.0) {
        double target = u * whole;
        const int c = vf_block_place(a.chunks, target, sh, piece);
        got = vf_block_entry(c, a.V, target, sh, [&](int i) {
          return fmax(vf_weight(vf_clean(row[i]), of_p.top, scale, sh.table) * inv - vf_weight(vf_clean(row_q[i]), of_q.top, scale, sh.table) * inv_q, 0.0);
        });
      }
    }
    if (got < 0 && sum > 0.0) {
      double target = u * sum;
      const int c = vf_block_place(a.chunks, target, sh, [&](int i) { return s_part[i]; });
      got = vf_block_entry(c, a.V, target, sh, [&](int i) { return vf_weight(vf_clean(row[i]), of_p.top, scale, sh.table); });
    }
    got = max(got, 0);
  }
  for (int j = tid; j < a.width; j += kVfThreads) {
    out[j] = j < kept ? a.tokens[t0 + j + 1] : j == kept ? got : -1;
    path[j] = j <= kept ? j : -1;
  }
  if (tid == 0) a.count[s] = kept + 1;
  pdl_arrived();
}

}  // namespace pmm

// Bytes of scratch for `rows` rows of V entries.
PMM_EXPORT long long pmm_verify_scratch(long long rows, int V) {
  const long long chunks = (V + pmm::kVfChunk - 1) / pmm::kVfChunk;
  return 2 * rows * chunks * static_cast<long long>(sizeof(pmm::VfChunk)) + rows * 4;
}

PMM_EXPORT int pmm_verify_drafts(const float* logits, long long ld, const float* draft, long long ld_draft, const int* tokens, const int* parents,
                                 const int* cu, int n, const float* uniforms, const float* temperature, int V, int n_rows, void* scratch,
                                 int* tokens_out, int* path, int width, int* count, int sms, cudaStream_t stream) {
  if (n <= 0) return 0;
  const int chunks = V > 0 ? (V + pmm::kVfChunk - 1) / pmm::kVfChunk : 0;
  if (V <= 0 || sms < 1 || chunks > pmm::kVfChunksMax || n_rows < 0 || static_cast<long long>(n_rows) * chunks > 0x3fffffffll || width <= 0 || !scratch || reinterpret_cast<uintptr_t>(scratch) % 16 ||
      (draft && parents) || n > 0x7fffffff / pmm::kVfCluster)
    return PMM_ERR_BAD_ARGUMENT;
  // Requests are read and written side by side.
  const long long out_bytes = 4ll * n * width, rows_bytes = 4ll * n_rows;
  const pmm::Extent written[] = {{tokens_out, out_bytes}, {path, out_bytes}, {count, 4ll * n}, {scratch, pmm_verify_scratch(n_rows, V)}};
  const pmm::Extent read[] = {{tokens, rows_bytes}, {parents, rows_bytes}, {uniforms, rows_bytes}, {cu, 4ll * (n + 1)}, {temperature, 4ll * n}};
  if (pmm::overlap(written, read)) return PMM_ERR_OVERLAP;
  for (int i = 0; i < 4; ++i) {
    for (int j = 0; j < i; ++j)
      if (pmm::overlap(written[i].at, written[i].bytes, written[j].at, written[j].bytes)) return PMM_ERR_OVERLAP;
    if (pmm::rows_overlap(logits, n_rows, 4 * ld, 4ll * V, written[i].at, written[i].bytes) ||
        pmm::rows_overlap(draft, n_rows, 4 * ld_draft, 4ll * V, written[i].at, written[i].bytes))
      return PMM_ERR_OVERLAP;
  }
  pmm::VerifyArgs a{};
  a.logits = logits;
  a.ld = ld;
  a.draft = draft;
  a.ld_draft = ld_draft;
  a.tokens = tokens;
  a.parents = parents;
  a.cu = cu;
  a.n = n;
  a.uniforms = uniforms;
  a.temperature = temperature;
  a.V = V;
  a.n_rows = n_rows;
  a.chunks = chunks;
  a.stats = static_cast<pmm::VfChunk*>(scratch);
  a.drawn = reinterpret_cast<int*>(a.stats + 2 * static_cast<size_t>(n_rows) * chunks);
  a.tokens_out = tokens_out;
  a.path = path;
  a.width = width;
  a.count = count;
  const unsigned blocks = (static_cast<unsigned>(chunks) * n_rows + pmm::kVfWarps - 1) / pmm::kVfWarps;
  if (n_rows > 0)
    pmm::launch_pdl(draft ? pmm::verify_stats_kernel<false> : pmm::verify_stats_kernel<true>, dim3(blocks, draft ? 2 : 1), dim3(pmm::kVfThreads), 0, stream, a);
  const size_t smem = draft ? 4 * static_cast<size_t>(chunks) * sizeof(double) : 0;
  if (smem > 16 * 1024) {  // (a vocabulary of half a million; attributes hold for the current device: set at every call)
    const cudaError_t e = cudaFuncSetAttribute(pmm::verify_walk_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return static_cast<int>(e);
  }
  // as many blocks a request as are on the device at once (two a multiprocessor), up to 16: 64 chains at 130,049 take 97 us with four, 105
  // with eight, 118 with two; 16 trees of 16 nodes at 65,537 22 with 16, 25 with eight, 31 with four
  a.cluster = pmm::kVfCluster;
  while (a.cluster > 1 && static_cast<long long>(n) * a.cluster > 2ll * sms) a.cluster /= 2;
  if (a.cluster > 8) {
    const cudaError_t e = cudaFuncSetAttribute(pmm::verify_walk_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return static_cast<int>(e);
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(n) * a.cluster);
  cfg.blockDim = dim3(pmm::kVfThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attrs[2];
  attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[0].val.programmaticStreamSerializationAllowed = 1;
  attrs[1].id = cudaLaunchAttributeClusterDimension;
  attrs[1].val.clusterDim.x = a.cluster;
  attrs[1].val.clusterDim.y = 1;
  attrs[1].val.clusterDim.z = 1;
  cfg.attrs = attrs;
  cfg.numAttrs = 2;
  cudaLaunchKernelEx(&cfg, pmm::verify_walk_kernel, a);
  return pmm::launch_status();
}
