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
// thousand would come out differently from the formula, so weights, sums and comparisons are in 64 bits.
// First launch: a block per (row, 4,096 entries) reads its entries once and leaves their maximum, its place and the sum of
// exp((l - maximum) / T).  Second launch: a cluster of eight blocks per request.
#include "common.cuh"
#include <math_constants.h>

namespace pmm {

constexpr int kVfThreads = 256;
constexpr int kVfEach = 16;
constexpr int kVfChunk = kVfThreads * kVfEach;
constexpr int kVfCluster = 8;
constexpr int kVfChunksMax = 1024;  // chunk sums of a row in shared memory
constexpr int kVfStride = kVfEach + 1;  // (a thread's entries of a chunk side by side, threads in different banks)

struct VfChunk {
  double sum;   // of exp((l - top) / T)
  float top;
  int at;       // the first index that holds top
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
};

// The request that row r belongs to: how many end at or before it.  Called by the whole block.
__device__ __forceinline__ int vf_request(const int* cu, int n, int r) {
  int s = 0;
  for (int b = 0; b < n; b += kVfThreads) {
    const int i = b + static_cast<int>(threadIdx.x);
    const int c = __syncthreads_count(i < n && cu[i + 1] <= r);
    s += c;
    if (c < kVfThreads) break;
  }
  return s;
}

__device__ __forceinline__ float vf_clean(float l) { return l == l ? l : -CUDART_INF_F; }

// exp((l - top) / T) as the formulas above want it at infinities.
__device__ __forceinline__ double vf_weight(float l, float top, double inv_t) {
  if (l == top) return top == -CUDART_INF_F ? 0.0 : 1.0;
  if (l == -CUDART_INF_F || top == CUDART_INF_F) return 0.0;
  return exp((static_cast<double>(l) - static_cast<double>(top)) * inv_t);
}

__global__ void __launch_bounds__(kVfThreads) verify_stats_kernel(const VerifyArgs a) {
  __shared__ float s_top[kVfThreads / 32];
  __shared__ int s_at[kVfThreads / 32];
  __shared__ double s_sum[kVfThreads / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int r = blockIdx.x / a.chunks, c = blockIdx.x % a.chunks, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const bool of_draft = blockIdx.y == 1;
  if (r >= a.cu[a.n]) return;
  const int s = vf_request(a.cu, a.n, r);
  const float temp = a.temperature ? a.temperature[s] : 0.f;
  const bool greedy = !(temp > 0.f);
  if (of_draft && (greedy || r == a.cu[s + 1] - 1)) return;  // (nothing was drafted behind a chain's last token)
  const float* row = of_draft ? a.draft + r * a.ld_draft : a.logits + r * a.ld;
  const int base = c * kVfChunk;
  float v[kVfEach];
#pragma unroll
  for (int k = 0; k < kVfEach; ++k) {
    const int i = base + k * kVfThreads + tid;
    v[k] = i < a.V ? vf_clean(row[i]) : -CUDART_INF_F;
  }
  float top = v[0];
  int at = base + tid;
#pragma unroll
  for (int k = 1; k < kVfEach; ++k)
    if (v[k] > top) {
      top = v[k];
      at = base + k * kVfThreads + tid;
    }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float ot = __shfl_xor_sync(0xffffffffu, top, o);
    const int oa = __shfl_xor_sync(0xffffffffu, at, o);
    if (ot > top || (ot == top && oa < at)) {
      top = ot;
      at = oa;
    }
  }
  if (lane == 0) {
    s_top[warp] = top;
    s_at[warp] = at;
  }
  __syncthreads();
  top = s_top[0];
  at = s_at[0];
#pragma unroll
  for (int w = 1; w < kVfThreads / 32; ++w)
    if (s_top[w] > top || (s_top[w] == top && s_at[w] < at)) {
      top = s_top[w];
      at = s_at[w];
    }
  double sum = 0.0;
  if (!greedy) {
    const double inv_t = 1.0 / static_cast<double>(temp);
#pragma unroll
    for (int k = 0; k < kVfEach; ++k) sum += vf_weight(v[k], top, inv_t);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) s_sum[warp] = sum;
    __syncthreads();
    sum = 0.0;
#pragma unroll
    for (int w = 0; w < kVfThreads / 32; ++w) sum += s_sum[w];
  }
  if (tid == 0) a.stats[(static_cast<size_t>(of_draft ? a.n_rows : 0) + r) * a.chunks + c] = VfChunk{sum, top, at};
}

// A row's maximum (and its first place), and the sum of exp((l - maximum) / T) over the row, by one warp.
__device__ __forceinline__ void vf_row(const VfChunk* st, int chunks, double inv_t, float& top, int& at, double& sum) {
  const int lane = threadIdx.x & 31;
  top = -CUDART_INF_F;
  at = 0;
  for (int c = lane; c < chunks; c += 32)
    if (st[c].top > top) {
      top = st[c].top;
      at = st[c].at;
    }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float ot = __shfl_xor_sync(0xffffffffu, top, o);
    const int oa = __shfl_xor_sync(0xffffffffu, at, o);
    if (ot > top || (ot == top && oa < at)) {
      top = ot;
      at = oa;
    }
  }
  sum = 0.0;
  for (int c = lane; c < chunks; c += 32) sum += st[c].sum * vf_weight(st[c].top, top, inv_t);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}

// The first index of a chunk whose running sum of weight(i) passes `target` (the last with any weight where rounding leaves none).
// Called by the whole block; w: shared memory for the chunk's weights, scan for a double per warp.
template <typename W>
__device__ __forceinline__ int vf_pick(int base, int V, double target, W weight, double* w, double* scan, int* s_pick) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
#pragma unroll
  for (int k = 0; k < kVfEach; ++k) {
    const int i = base + k * kVfThreads + tid;
    const int e = k * kVfThreads + tid;
    w[e / kVfEach * kVfStride + e % kVfEach] = i < V ? weight(i) : 0.0;
  }
  if (tid == 0) {
    s_pick[0] = 0x7fffffff;
    s_pick[1] = -1;
  }
  __syncthreads();
  double own = 0.0;
  int last = -1;
#pragma unroll
  for (int k = 0; k < kVfEach; ++k) {
    const double x = w[tid * kVfStride + k];
    own += x;
    if (x > 0.0) last = tid * kVfEach + k;
  }
  double run = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double up = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += up;
  }
  if (lane == 31) scan[warp] = run;
  __syncthreads();
  double before = run - own;
  for (int i = 0; i < warp; ++i) before += scan[i];
  int found = 0x7fffffff;
  double at = before;
  for (int k = 0; k < kVfEach; ++k) {
    const double x = w[tid * kVfStride + k];
    at += x;
    if (x > 0.0 && at > target && found == 0x7fffffff) found = tid * kVfEach + k;
  }
  if (found != 0x7fffffff) atomicMin(&s_pick[0], found);
  if (last >= 0) atomicMax(&s_pick[1], last);
  __syncthreads();
  return base + (s_pick[0] != 0x7fffffff ? s_pick[0] : max(s_pick[1], 0));
}

// The chunk in which the running sum of part[0 .. chunks) passes `target` (the last with any weight where rounding leaves none),
// and what of the target is left in it.  Every thread walks by itself.
__device__ __forceinline__ int vf_chunk(const double* part, int chunks, double& target) {
  double run = 0.0;
  int last = 0;
  double before_last = 0.0;
  for (int c = 0; c < chunks; ++c) {
    if (part[c] > 0.0) {
      if (run + part[c] > target) {
        target -= run;
        return c;
      }
      last = c;
      before_last = run;
    }
    run += part[c];
  }
  target -= before_last;
  return last;
}

__global__ void __launch_bounds__(kVfThreads) __cluster_dims__(kVfCluster, 1, 1) verify_walk_kernel(const VerifyArgs a) {
  __shared__ double s_w[kVfThreads * kVfStride];
  __shared__ double s_part[kVfChunksMax];
  __shared__ double s_scan[kVfThreads / 32];
  __shared__ int s_pick[2];
  __shared__ float s_top[2];
  __shared__ double s_total[2];
  __shared__ int s_best, s_kept;
  pdl_wait();
  const int s = blockIdx.x / kVfCluster, rank = blockIdx.x % kVfCluster, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int t0 = a.cu[s], t1 = min(a.cu[s + 1], a.n_rows);
  const int nodes = t1 - t0;
  const float temp = a.temperature ? a.temperature[s] : 0.f;
  const bool greedy = !(temp > 0.f);
  const double inv_t = greedy ? 1.0 : 1.0 / static_cast<double>(temp);
  int* out = a.tokens_out + static_cast<size_t>(s) * a.width;
  int* path = a.path + static_cast<size_t>(s) * a.width;
  if (nodes <= 0) {  // (the same for the whole cluster)
    if (rank == 0) {
      for (int j = tid; j < a.width; j += kVfThreads) out[j] = path[j] = -1;
      if (tid == 0) a.count[s] = 0;
    }
    return;
  }
  auto stats = [&](int r, bool of_draft) { return a.stats + (static_cast<size_t>(of_draft ? a.n_rows : 0) + r) * a.chunks; };
  // a row's chunk sums against its maximum into s_part, maximum and total into place `k`, the place of the maximum into s_best
  auto row_parts = [&](int r, bool of_draft, int k, bool parts) {
    const VfChunk* st = stats(r, of_draft);
    if (warp == 0) {
      float top;
      int at;
      double sum;
      vf_row(st, a.chunks, inv_t, top, at, sum);
      if (lane == 0) {
        s_top[k] = top;
        s_total[k] = sum;
        if (k == 0) s_best = at;
      }
    }
    __syncthreads();
    if (parts)
      for (int c = tid; c < a.chunks; c += kVfThreads) s_part[c] = st[c].sum * vf_weight(st[c].top, s_top[k], inv_t);
    __syncthreads();
  };
  // a draw from p of row r with u, by one block (-1: no token has any weight)
  auto draw = [&](int r, float u) {
    row_parts(r, false, 0, !greedy);
    int got = s_best;
    if (!greedy && s_total[0] > 0.0) {
      double whole = 0.0;
      for (int c = 0; c < a.chunks; ++c) whole += s_part[c];
      double target = static_cast<double>(u) * whole;
      const int c = vf_chunk(s_part, a.chunks, target);
      const float* row = a.logits + r * a.ld;
      const float top = s_top[0];
      got = vf_pick(c * kVfChunk, a.V, target, [&](int i) { return vf_weight(vf_clean(row[i]), top, inv_t); }, s_w, s_scan, s_pick);
    }
    if (s_top[0] == -CUDART_INF_F) got = -1;
    __syncthreads();
    return got;
  };

  if (a.draft == nullptr) {
    // ---- fixed proposals: every node's draw, the blocks of the cluster side by side; then the walk
    for (int i = rank; i < nodes; i += kVfCluster) {
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
    return;
  }

  // ---- a chain from a draft's distribution: which tokens are kept (every block of the cluster finds out for itself)
  const int drafted = min(nodes, a.width) - 1;
  if (tid == 0) s_kept = drafted;
  __syncthreads();
  for (int i = 1 + warp; i <= drafted; i += kVfThreads / 32) {
    const int r = t0 + i - 1, x = a.tokens[t0 + i];
    float top, top_q = 0.f;
    int at, at_q;
    double sum, sum_q = 0.0;
    vf_row(stats(r, false), a.chunks, inv_t, top, at, sum);
    bool ok = false;
    if (greedy) {
      ok = at == x && top > -CUDART_INF_F;
    } else if (x >= 0 && x < a.V) {
      vf_row(stats(r, true), a.chunks, inv_t, top_q, at_q, sum_q);
      const double p = vf_weight(vf_clean(a.logits[r * a.ld + x]), top, inv_t), q = vf_weight(vf_clean(a.draft[r * a.ld_draft + x]), top_q, inv_t);
      // u q / sum_q < p / sum (a draft without weight anywhere proposes nothing that could be kept)
      ok = sum > 0.0 && sum_q > 0.0 && static_cast<double>(a.uniforms[t0 + i]) * (q / sum_q) < p / sum;
    }
    if (!ok && lane == 0) atomicMin(&s_kept, i - 1);
  }
  __syncthreads();
  const int kept = s_kept;
  const int r = t0 + kept;
  const float u = a.uniforms[t0];
  const bool rest = !greedy && kept < drafted;   // a draft was refused: what p has more than q
  int got = -1;
  if (rest) {
    row_parts(r, false, 0, false);
    row_parts(r, true, 1, false);
    const float* row = a.logits + r * a.ld;
    const float* row_q = a.draft + r * a.ld_draft;
    const float top = s_top[0], top_q = s_top[1];
    const double inv = s_total[0] > 0.0 ? 1.0 / s_total[0] : 0.0, inv_q = s_total[1] > 0.0 ? 1.0 / s_total[1] : 0.0;
    auto weight = [&](int i) {
      const double p = vf_weight(vf_clean(row[i]), top, inv_t) * inv, q = vf_weight(vf_clean(row_q[i]), top_q, inv_t) * inv_q;
      return fmax(p - q, 0.0);
    };
    cluster_sync();  // (every block of the cluster is there: its shared memory may be written)
    for (int c = rank; c < a.chunks; c += kVfCluster) {
      double sum = 0.0;
#pragma unroll 4
      for (int k = 0; k < kVfEach; ++k) {
        const int i = c * kVfChunk + k * kVfThreads + tid;
        if (i < a.V) sum += weight(i);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane == 0) s_scan[warp] = sum;
      __syncthreads();
      if (tid < kVfCluster) {  // the chunk's sum to every block of the cluster
        sum = 0.0;
        for (int w = 0; w < kVfThreads / 32; ++w) sum += s_scan[w];
        unsigned dst;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(dst) : "r"(static_cast<unsigned>(__cvta_generic_to_shared(&s_part[c]))), "r"(tid));
        asm volatile("st.shared::cluster.f64 [%0], %1;\n" ::"r"(dst), "d"(sum) : "memory");
      }
      __syncthreads();
    }
    cluster_sync();
    double whole = 0.0;
    for (int c = 0; c < a.chunks; ++c) whole += s_part[c];
    if (whole > 0.0) {
      double target = static_cast<double>(u) * whole;
      const int c = vf_chunk(s_part, a.chunks, target);
      if (c % kVfCluster != rank) return;
      got = vf_pick(c * kVfChunk, a.V, target, weight, s_w, s_scan, s_pick);
    } else if (rank != 0) {
      return;
    }
    __syncthreads();
  } else if (rank != 0) {
    return;
  }
  if (got < 0) got = max(draw(r, u), 0);
  for (int j = tid; j < a.width; j += kVfThreads) {
    out[j] = j < kept ? a.tokens[t0 + j + 1] : j == kept ? got : -1;
    path[j] = j <= kept ? j : -1;
  }
  if (tid == 0) a.count[s] = kept + 1;
}

}  // namespace pmm

// Bytes of scratch for `rows` rows of V entries.
PMM_EXPORT long long pmm_verify_scratch(long long rows, int V) {
  const long long chunks = (V + pmm::kVfChunk - 1) / pmm::kVfChunk;
  return 2 * rows * chunks * static_cast<long long>(sizeof(pmm::VfChunk)) + rows * 4;
}

PMM_EXPORT int pmm_verify_drafts(const float* logits, long long ld, const float* draft, long long ld_draft, const int* tokens, const int* parents,
                                 const int* cu, int n, const float* uniforms, const float* temperature, int V, int n_rows, void* scratch,
                                 int* tokens_out, int* path, int width, int* count, cudaStream_t stream) {
  if (n <= 0) return 0;
  const int chunks = V > 0 ? (V + pmm::kVfChunk - 1) / pmm::kVfChunk : 0;
  if (V <= 0 || chunks > pmm::kVfChunksMax || n_rows < 0 || static_cast<long long>(n_rows) * chunks > 0x7fffffffll || width <= 0 || !scratch || reinterpret_cast<uintptr_t>(scratch) % 16 ||
      (draft && parents) || n > 0x7fffffff / pmm::kVfCluster)
    return PMM_ERR_BAD_ARGUMENT;
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
  if (n_rows > 0)
    pmm::launch_pdl(pmm::verify_stats_kernel, dim3(chunks * n_rows, draft ? 2 : 1), dim3(pmm::kVfThreads), 0, stream, a);
  pmm::launch_pdl(pmm::verify_walk_kernel, dim3(n * pmm::kVfCluster), dim3(pmm::kVfThreads), 0, stream, a);
  return pmm::launch_status();
}
