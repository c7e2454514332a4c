// Attention of drafted tokens over a paged cache: token i of request s sees the request's held[s] cached keys (the last
// `window` positions up to its own, where there is a window) and, among the request's own tokens of this step, those whose
// bits its mask holds (without masks: those in front of it, and itself), with `window_step` only as far as the window reaches.
//   sc[j] = (q.K[j]) * scale;  p = exp(sc - max);  o = sum p V / sum p,   0 for a row that sees no key
// The step's own keys and values lie densely in k and v: the cache takes only those that are kept in the end.
//
// Float arithmetic on the CUDA cores, any storage type and head size, in two kernels: up to a head size of 256 blocks of rows (a row: a
// token and a query head of the group) that share what they read of the keys, beyond it a block per token and query head.
#include "tree_attention.cuh"
#include <math_constants.h>

#include <type_traits>

namespace pmm {

constexpr int kTaWarps = 8;

template <typename S>
struct TreeAttnArgs {
  const S* q;
  long long ldq;
  const S* k;
  long long ldk;
  const S* v;
  long long ldv;
  const S* pool;
  const int* block_table;
  int max_blocks;
  int pages;
  const int* held;
  const int* cu;
  const int* positions;            // [T], where there is a window
  const unsigned long long* mask;  // [T, words] or nullptr: causal
  int words;
  const float* sink;               // [Hq] or nullptr
  S* out;
  float scale;
  int window;
  int window_step;                 // the window limits the step's own tokens too, by their positions
  int page_size, n_seq, Hq, Hkv, Dh;
};

__device__ __forceinline__ float ta_dot(const float* qw, const float* kr, int Dh) {
  float dot = 0.f;
#pragma unroll 8
  for (int d = 0; d < Dh; d += 4) {
    const float4 x = ldf4(kr + d);
    dot += qw[d] * x.x;
    dot += qw[d + 1] * x.y;
    dot += qw[d + 2] * x.z;
    dot += qw[d + 3] * x.w;
  }
  return dot;
}
__device__ __forceinline__ float ta_dot(const float* qw, const __nv_bfloat16* kr, int Dh) {
  float dot = 0.f;
#pragma unroll 8
  for (int d = 0; d < Dh; d += 8) {
    const uint4 raw = *reinterpret_cast<const uint4*>(kr + d);
    const __nv_bfloat162* h2 = reinterpret_cast<const __nv_bfloat162*>(&raw);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __bfloat1622float2(h2[i]);
      dot += qw[d + 2 * i] * f.x;
      dot += qw[d + 2 * i + 1] * f.y;
    }
  }
  return dot;
}

// Whether bit j of a token's mask is set.
__device__ __forceinline__ bool ta_sees(const unsigned long long* mask, int words, int j) {
  return j < 64 * words && (mask[j >> 6] >> (j & 63) & 1ull) != 0ull;
}

// Head sizes beyond 256.  A block per (token, query head); its eight warps share the keys in pieces of 32 (a key per lane for the scores, a
// slice of the head per lane for the values) and merge their maxima, sums and results at the end.
template <typename S, int ACC>
__global__ void __launch_bounds__(kTaWarps * 32, 3) tree_attention_kernel(const TreeAttnArgs<S> a, int T) {
  extern __shared__ float qs[];  // the query, then every warp's result
  __shared__ float s_m[kTaWarps], s_l[kTaWarps];
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int t = blockIdx.x, hq = blockIdx.y, Dh = a.Dh;
  if (t >= a.cu[a.n_seq]) return;
  int seq = 0;
  for (int b = 0; b < a.n_seq; b += kTaWarps * 32) {
    const int c = __syncthreads_count(b + tid < a.n_seq && a.cu[b + tid + 1] <= t);
    seq += c;
    if (c < kTaWarps * 32) break;
  }
  const int hk = hq / (a.Hq / a.Hkv);
  // (bounds may pass the step's rows: those that are not there are not read)
  const int t0 = min(max(a.cu[seq], 0), T), n_new = min(max(a.cu[seq + 1], t0), T) - t0;
  const int held = max(0, static_cast<int>(min(static_cast<long long>(a.held[seq]), static_cast<long long>(a.max_blocks) * a.page_size)));
  const int lo = a.window != 0 ? first_visible(a.positions[t], a.window) : 0;
  const int* bt = a.block_table + static_cast<size_t>(seq) * a.max_blocks;
  const unsigned long long* mask = a.mask ? a.mask + static_cast<size_t>(t) * a.words : nullptr;
  const long long kv_dim = static_cast<long long>(a.Hkv) * Dh;
  const long long v_plane = a.page_size * kv_dim;
  const S* q = a.q + t * a.ldq + hq * Dh;
  for (int d = tid; d < Dh; d += kTaWarps * 32) qs[d] = ldf(q + d);
  __syncthreads();

  float m = -CUDART_INF_F, l = 0.f, acc[ACC];
#pragma unroll
  for (int i = 0; i < ACC; ++i) acc[i] = 0.f;
  for (int part = 0; part < 2; ++part) {  // the cache, then the step's own tokens
    const int begin = part == 0 ? lo : 0, end = part == 0 ? held : n_new;
    for (int base = begin + warp * 32; base < end; base += kTaWarps * 32) {
      const int j = base + lane;
      const bool valid = j < end && (part == 0 || ((mask ? ta_sees(mask, a.words, j) : j <= t - t0) && (!a.window_step || a.positions[t0 + j] >= lo)));
      const S *kr = nullptr, *vr = nullptr;
      float sc = -CUDART_INF_F;
      if (valid) {
        if (part == 0) {
          const int page = min(max(bt[j / a.page_size], 0), a.pages - 1);  // (no read leaves the pool)
          kr = a.pool + (static_cast<long long>(page) * 2 * a.page_size + j % a.page_size) * kv_dim + hk * Dh;
          vr = kr + v_plane;
        } else {
          kr = a.k + (t0 + j) * a.ldk + hk * Dh;
          vr = a.v + (t0 + j) * a.ldv + hk * Dh;
        }
        sc = ta_dot(qs, kr, Dh) * a.scale;
      }
      const unsigned left = __ballot_sync(0xffffffffu, valid);
      if (left == 0) continue;
      const float m_new = fmaxf(m, warp_max(sc));
      const float mu = m_new == -CUDART_INF_F ? 0.f : m_new;
      const float p = valid ? expf(sc - mu) : 0.f;
      const float corr = expf(m - mu);
      m = m_new;
      l = l * corr + warp_sum(p);
#pragma unroll
      for (int i = 0; i < ACC; ++i) acc[i] *= corr;
      // values of kKeys keys at a time, so that as many rows travel together; of keys that are not seen they may be anything
      constexpr int kKeys = 32 / ACC;
#pragma unroll 1
      for (int b = 0; b < 32; b += kKeys) {
        const unsigned some = left >> b & ((1u << kKeys) - 1u);
        if (some == 0) continue;
        float x[kKeys][ACC], pj[kKeys];
#pragma unroll
        for (int u = 0; u < kKeys; ++u) {
          pj[u] = __shfl_sync(0xffffffffu, p, b + u);
          const S* row = reinterpret_cast<const S*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(vr), b + u));
#pragma unroll
          for (int i = 0; i < ACC; ++i) {
            const int d = lane + 32 * i;
            x[u][i] = (some >> u & 1u) && d < Dh ? ldf(row + d) : 0.f;
          }
        }
#pragma unroll
        for (int u = 0; u < kKeys; ++u)
#pragma unroll
          for (int i = 0; i < ACC; ++i) acc[i] += pj[u] * x[u][i];
      }
    }
  }
  if (a.sink && warp == 0) {  // a score without key or value that counts once (of -inf: not at all)
    const float m_new = fmaxf(m, a.sink[hq]), mu = m_new == -CUDART_INF_F ? 0.f : m_new;
    const float corr = expf(m - mu);
    l = l * corr + expf(a.sink[hq] - mu);
#pragma unroll
    for (int i = 0; i < ACC; ++i) acc[i] *= corr;
    m = m_new;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < ACC; ++i) {
    const int d = lane + 32 * i;
    if (d < Dh) qs[warp * Dh + d] = acc[i];
  }
  if (lane == 0) {
    s_m[warp] = m;
    s_l[warp] = l;
  }
  __syncthreads();
  float top = s_m[0];
#pragma unroll
  for (int w = 1; w < kTaWarps; ++w) top = fmaxf(top, s_m[w]);
  if (top == -CUDART_INF_F) top = 0.f;
  float f[kTaWarps], sum = 0.f;
#pragma unroll
  for (int w = 0; w < kTaWarps; ++w) {
    f[w] = expf(s_m[w] - top);
    sum += s_l[w] * f[w];
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;  // (NaN stays NaN)
  for (int d = tid; d < Dh; d += kTaWarps * 32) {
    float o = 0.f;
#pragma unroll
    for (int w = 0; w < kTaWarps; ++w) o += s_l[w] != 0.f ? qs[w * Dh + d] * f[w] : 0.f;
    stf(a.out + (static_cast<long long>(t) * a.Hq + hq) * Dh + d, o * inv);
  }
}

// Head sizes up to 256.  A cluster of blocks takes up to 32 rows of one request and key/value head; its blocks take the keys in tiles of 64 in
// turn.  A tile of K and V lies in shared memory once for all rows (with a block per row, as beyond 256, 8 requests of up to 19 tokens, 32 / 8
// heads of 128, over up to 433 keys took 123 us, so 55).  A warp has up to eight rows and 32 of a tile's keys: a lane a key for the
// scores, a slice of the head a lane for the values, so maxima, sums and results stay in its registers.  In the end every block leaves
// (maximum, sum, unnormalised result) in its shared memory, and the cluster's blocks join a share of the rows each, in the order of the
// blocks.  What bounds it: shared memory, 12 reads of 128 bytes for 32 products of a warp's scores, 24 for 128 of its values, and one tile at
// a time, so that copies and products do not overlap: 14 requests of 5 over 2,340 keys, 32 / 8 heads of 128 in float32, take 262 us where
// the keys' bytes are 41; shared memory is busy for 42 % of the time there, the float units for 29.
constexpr int kTfRows = 32, kTfKeys = 64, kTfThreads = 256, kTfPer = 8;
constexpr int kTfCluster = 8;  // blocks of a cluster at most

// Bytes of shared memory: the queries; a tile of K and V, rows 16 bytes further apart than they are long (in the end two parts of the results).
__host__ __device__ constexpr int tf_row(int dh, int elem) { return dh * elem + 16; }
__host__ __device__ constexpr size_t tf_smem(int dh, int elem) {
  return static_cast<size_t>(kTfRows) * dh * sizeof(float) + static_cast<size_t>(2) * kTfKeys * tf_row(dh, elem);
}
static_assert(2 * kTfKeys * 2 >= 2 * kTfRows * 4, "two parts of float results fit where a tile of two-byte elements was");
__device__ __forceinline__ void tf_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
// A float of block `rank`'s shared memory, where this block has it at p.
__device__ __forceinline__ float tf_remote(const float* p, int rank) {
  unsigned at;
  float x;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(at) : "r"(static_cast<unsigned>(__cvta_generic_to_shared(p))), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];\n" : "=f"(x) : "r"(at) : "memory");
  return x;
}
// s[i] += q[i] . k over the head, for N rows.
template <int N>
__device__ __forceinline__ void tf_scores(float (&s)[N], const float* const (&q)[N], const float* kr, int Dh) {
#pragma unroll 2
  for (int d = 0; d < Dh; d += 4) {
    const float4 x = *reinterpret_cast<const float4*>(kr + d);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float4 y = *reinterpret_cast<const float4*>(q[i] + d);
      s[i] += y.x * x.x;
      s[i] += y.y * x.y;
      s[i] += y.z * x.z;
      s[i] += y.w * x.w;
    }
  }
}
template <int N>
__device__ __forceinline__ void tf_scores(float (&s)[N], const float* const (&q)[N], const __nv_bfloat16* kr, int Dh) {
  for (int d = 0; d < Dh; d += 8) {
    const uint4 raw = *reinterpret_cast<const uint4*>(kr + d);
    const __nv_bfloat162* h2 = reinterpret_cast<const __nv_bfloat162*>(&raw);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const float2 x0 = __bfloat1622float2(h2[2 * c]), x1 = __bfloat1622float2(h2[2 * c + 1]);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float4 y = *reinterpret_cast<const float4*>(q[i] + d + 4 * c);
        s[i] += y.x * x0.x;
        s[i] += y.y * x0.y;
        s[i] += y.z * x1.x;
        s[i] += y.w * x1.y;
      }
    }
  }
}

// STEP: the window limits the step's own tokens too (in a form of its own: asked of every row it costs the others 3 %).
template <typename S, int ACC, bool STEP>
__global__ void __launch_bounds__(kTfThreads, ACC <= 4 ? 2 : 1) tree_rows_kernel(const TreeAttnArgs<S> a, int T, int cluster) {
  extern __shared__ __align__(16) unsigned char tf_mem[];
  __shared__ float2 s_ml[2][kTfRows];
  __shared__ __align__(16) float s_p[kTfThreads / 32][kTfPer][32];
  __shared__ int s_sum[kTfThreads / 32], s_found[2], s_tok[kTfRows], s_lo[kTfRows];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, Dh = a.Dh, G = a.Hq / a.Hkv;
  const int tile = blockIdx.x / cluster, rank = blockIdx.x % cluster, hk = blockIdx.y;
  pdl_launch_dependents();
  pdl_wait();
  // ---- the request whose row tile this is
  if (tid == 0) s_found[0] = -1;
  int before = 0;
  for (int base = 0; base < a.n_seq; base += kTfThreads) {
    const int s = base + tid;
    int n = 0;
    if (s < a.n_seq) {
      const int b0 = min(max(a.cu[s], 0), T), b1 = min(max(a.cu[s + 1], b0), T);
      n = ((b1 - b0) * G + kTfRows - 1) / kTfRows;
    }
    int run = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += up;
    }
    if (lane == 31) s_sum[warp] = run;
    __syncthreads();
    int at = before;
#pragma unroll
    for (int w = 0; w < kTfThreads / 32; ++w) {
      if (w < warp) at += s_sum[w];
      before += s_sum[w];
    }
    at += run - n;
    if (tile >= at && tile < at + n) {
      s_found[0] = s;
      s_found[1] = tile - at;
    }
    __syncthreads();
    if (s_found[0] >= 0) break;
  }
  if (s_found[0] < 0) return;  // (the same for the whole cluster)
  const int seq = s_found[0], row0 = s_found[1] * kTfRows;
  const int t0 = min(max(a.cu[seq], 0), T), n_new = min(max(a.cu[seq + 1], t0), T) - t0;
  const int held = max(0, static_cast<int>(min(static_cast<long long>(a.held[seq]), static_cast<long long>(a.max_blocks) * a.page_size)));
  const int n_rows = min(kTfRows, n_new * G - row0);
  const int* bt = a.block_table + static_cast<size_t>(seq) * a.max_blocks;
  const long long kv_dim = static_cast<long long>(a.Hkv) * Dh, v_plane = a.page_size * kv_dim;
  float* sQ = reinterpret_cast<float*>(tf_mem);
  unsigned char* sK = tf_mem + static_cast<size_t>(kTfRows) * Dh * sizeof(float);
  const int row_bytes = tf_row(Dh, sizeof(S));
  unsigned char* sV = sK + kTfKeys * row_bytes;
  int first = 0;  // the first cached key that any of the rows may see (or the last one's end)
  if (a.window != 0) {
    first = held;
    for (int tok = row0 / G; tok <= (row0 + n_rows - 1) / G; ++tok) first = min(first, first_visible(a.positions[t0 + tok], a.window));
  }
  const int ctx_tiles = (held - first + kTfKeys - 1) / kTfKeys, n_tiles = ctx_tiles + (n_new + kTfKeys - 1) / kTfKeys;
  auto fetch = [&](int j) {  // four threads a key
    const bool own = j >= ctx_tiles;
    const int base = own ? (j - ctx_tiles) * kTfKeys : first + j * kTfKeys, key = tid >> 2;
    if (key < min(kTfKeys, (own ? n_new : held) - base)) {
      const S *kr, *vr;
      if (own) {
        kr = a.k + (t0 + base + key) * a.ldk + hk * Dh;
        vr = a.v + (t0 + base + key) * a.ldv + hk * Dh;
      } else {
        const int page = min(max(bt[(base + key) / a.page_size], 0), a.pages - 1);  // (no read leaves the pool)
        kr = a.pool + (static_cast<long long>(page) * 2 * a.page_size + (base + key) % a.page_size) * kv_dim + hk * Dh;
        vr = kr + v_plane;
      }
      const unsigned to = static_cast<unsigned>(__cvta_generic_to_shared(sK + key * row_bytes));
      constexpr int kElems = 16 / static_cast<int>(sizeof(S));
#pragma unroll 4
      for (int c = tid & 3; c < Dh / kElems; c += 4) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(to + 16 * c), "l"(kr + c * kElems) : "memory");
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(to + kTfKeys * row_bytes + 16 * c), "l"(vr + c * kElems) : "memory");
      }
    }
  };
  if (rank < n_tiles) {
    fetch(rank);
    for (int i = tid; i < n_rows * (Dh / 8); i += kTfThreads) {
      const int r = i / (Dh / 8), d = 8 * (i - r * (Dh / 8)), tok = (row0 + r) / G, h = (row0 + r) - tok * G;
      const S* from = a.q + (t0 + tok) * a.ldq + (hk * G + h) * Dh + d;
      const float4 x = ldf4(from), y = ldf4(from + 4);
      *reinterpret_cast<float4*>(sQ + r * Dh + d) = x;
      *reinterpret_cast<float4*>(sQ + r * Dh + d + 4) = y;
    }
  }
  if (tid < kTfRows) {
    const int tok = min(row0 + tid, n_new * G - 1) / G;
    s_tok[tid] = tok;
    s_lo[tid] = a.window != 0 ? first_visible(a.positions[t0 + tok], a.window) : 0;
  }
  const int half = warp >> 2, wr = warp & 3;                // of a tile's keys; of the rows: wr, wr + 4, ..
  const int mine = max(0, (n_rows - wr + 3) / 4);           // rows of this warp
  float m[kTfPer], l[kTfPer], acc[kTfPer][ACC];
#pragma unroll
  for (int i = 0; i < kTfPer; ++i) {
    m[i] = -CUDART_INF_F;
    l[i] = 0.f;
#pragma unroll
    for (int u = 0; u < ACC; ++u) acc[i][u] = 0.f;
  }
  for (int j = rank; j < n_tiles; j += cluster) {
    const bool own = j >= ctx_tiles;
    const int base = (own ? (j - ctx_tiles) * kTfKeys : first + j * kTfKeys) + 32 * half;
    const int n_keys = min(32, (own ? n_new : held) - base);  // of this warp's half
    asm volatile("cp.async.wait_all;\n" ::: "memory");
    __syncthreads();
    // N of the warp's rows, or more than it has: the last one again, whose results nobody reads (a question per row and step costs
    // more than its products)
    auto work = [&](auto rows) {
      constexpr int N = decltype(rows)::value;
      float s[N];
      const float* q[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        s[i] = 0.f;
        q[i] = sQ + (wr + 4 * min(i, mine - 1)) * Dh;
      }
      tf_scores<N>(s, q, reinterpret_cast<const S*>(sK + (32 * half + min(lane, n_keys - 1)) * row_bytes), Dh);
      unsigned sees[N];
      bool all = true;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int r = wr + 4 * min(i, mine - 1), tok = s_tok[r], key = base + lane;
        const bool see = lane < n_keys && (!own ? key >= s_lo[r] : a.mask ? ta_sees(a.mask + static_cast<size_t>(t0 + tok) * a.words, a.words, key) : key <= tok) &&
                         (!STEP || !own || a.positions[t0 + key] >= s_lo[r]);
        sees[i] = __ballot_sync(0xffffffffu, see);
        all = all && sees[i] == 0xffffffffu;
        const float sc = see ? s[i] * a.scale : -CUDART_INF_F;
        const float m_new = fmaxf(m[i], warp_max(sc)), mu = m_new == -CUDART_INF_F ? 0.f : m_new;
        const float corr = expf(m[i] - mu), p = see ? expf(sc - mu) : 0.f;  // (of a NaN: NaN)
        s_p[warp][i][lane] = p;
        m[i] = m_new;
        l[i] = l[i] * corr + p;  // (a lane's part of the sum)
#pragma unroll
        for (int u = 0; u < ACC; ++u) acc[i][u] *= corr;
      }
      __syncwarp();
      const unsigned char* vr = sV + 32 * half * row_bytes;
      auto value = [&](int k, int u) { return lane + 32 * u < Dh ? ldf(reinterpret_cast<const S*>(vr + k * row_bytes) + lane + 32 * u) : 0.f; };
      if (all) {
#pragma unroll 1
        for (int k = 0; k < 32; k += 4) {
          float v[4][ACC];
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int u = 0; u < ACC; ++u) v[e][u] = value(k + e, u);
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const float4 p = *reinterpret_cast<const float4*>(&s_p[warp][i][k]);
#pragma unroll
            for (int u = 0; u < ACC; ++u) {
              acc[i][u] += p.x * v[0][u];
              acc[i][u] += p.y * v[1][u];
              acc[i][u] += p.z * v[2][u];
              acc[i][u] += p.w * v[3][u];
            }
          }
        }
      } else {
#pragma unroll 2
        for (int k = 0; k < n_keys; ++k) {
          float v[ACC];
#pragma unroll
          for (int u = 0; u < ACC; ++u) v[u] = value(k, u);
#pragma unroll
          for (int i = 0; i < N; ++i)
            if (sees[i] >> k & 1u) {  // (values of keys that are not seen may be anything)
              const float p = s_p[warp][i][k];
#pragma unroll
              for (int u = 0; u < ACC; ++u) acc[i][u] += p * v[u];
            }
        }
      }
    };
    if (n_keys > 0) {
      if (mine > 4)
        work(std::integral_constant<int, 8>{});
      else if (mine > 2)
        work(std::integral_constant<int, 4>{});
      else if (mine == 2)
        work(std::integral_constant<int, 2>{});
      else if (mine == 1)
        work(std::integral_constant<int, 1>{});
    }
    __syncthreads();  // (the tile has been used)
    if (j + cluster < n_tiles) fetch(j + cluster);
  }
  // ---- every block's parts, then a share of the rows a block
  float* part = reinterpret_cast<float*>(sK);  // [half][rows][Dh]
#pragma unroll
  for (int i = 0; i < kTfPer; ++i) {
    if (i >= mine) continue;
    const int r = wr + 4 * i;
#pragma unroll
    for (int u = 0; u < ACC; ++u)
      if (lane + 32 * u < Dh) part[(half * kTfRows + r) * Dh + lane + 32 * u] = acc[i][u];
    const float sum = warp_sum(l[i]);
    if (lane == 0) s_ml[half][r] = make_float2(m[i], sum);
  }
  tf_cluster_sync();
  for (int r = rank + cluster * warp; r < n_rows; r += cluster * (kTfThreads / 32)) {
    const int tok = s_tok[r], hq = hk * G + (row0 + r) - tok * G;
    // (lane 2 c + h: half h of block c)
    const bool there = lane < 2 * cluster;
    const float part_m = there ? tf_remote(&s_ml[lane & 1][r].x, lane >> 1) : -CUDART_INF_F, part_l = there ? tf_remote(&s_ml[lane & 1][r].y, lane >> 1) : 0.f;
    float top = warp_max(part_m);
    if (a.sink) top = fmaxf(top, a.sink[hq]);  // a score without key or value that counts once
    if (top == -CUDART_INF_F) top = 0.f;
    const float f = expf(part_m - top);
    float sum = warp_sum(part_l * f);
    if (a.sink) sum += expf(a.sink[hq] - top);
    const float inv = sum == 0.f ? 0.f : 1.f / sum;  // (NaN stays NaN)
    const unsigned some = __ballot_sync(0xffffffffu, part_l != 0.f);  // (parts in which the row sees a key)
    float o[ACC];
#pragma unroll
    for (int u = 0; u < ACC; ++u) o[u] = 0.f;
#pragma unroll 1
    for (int p0 = 0; p0 < 2 * cluster; p0 += 4) {
      float x[4][ACC];
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int u = 0; u < ACC; ++u)
          x[e][u] = (some >> (p0 + e) & 1u) && lane + 32 * u < Dh ? tf_remote(part + (((p0 + e) & 1) * kTfRows + r) * Dh + lane + 32 * u, (p0 + e) >> 1) : 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float fp = __shfl_sync(0xffffffffu, f, p0 + e);
#pragma unroll
        for (int u = 0; u < ACC; ++u)
          if (some >> (p0 + e) & 1u) o[u] += fp * x[e][u];
      }
    }
    S* out = a.out + (static_cast<long long>(t0 + tok) * a.Hq + hq) * Dh;
#pragma unroll
    for (int u = 0; u < ACC; ++u)
      if (lane + 32 * u < Dh) stf(out + lane + 32 * u, o[u] * inv);
  }
  tf_cluster_sync();  // (no block leaves while another reads its parts)
}

template <typename S, int ACC>
int launch_tree_rows(const TreeAttnArgs<S>& a, int T, int sms, cudaStream_t stream) {
  const int G = a.Hq / a.Hkv;
  const long long tiles = (static_cast<long long>(T) * G + kTfRows - 1) / kTfRows + min(T, a.n_seq);  // (at most)
  // Blocks of a cluster: the tables' width tells how many tiles of keys there may be, and requests of equal size how many tiles of rows.  Up
  // to four blocks a multiprocessor, and from two on at least two tiles a block.  Float32, us with 1, 2, 4 and 8 blocks, the rule's in brackets:
  // 8 / 2 heads of 64: 1 request of 5 over 700 keys 73, 40, 23, [18]; 4 of 12 over 300 40, 23, [18], 15; 14 of 5 over 2,340 221, 129, 86, [48];
  // 64 of 4 over 500 49, 29, [36], 54; 100 of 2 over 200 20, [27], 31, 54; 32 / 8 heads of 128: 6 of 2 over 514 43, 32, [21], 29; 12 of 1 over
  // 53 11, [10], 16, 29; 19 of 8 over 608 145, [135], 121, 162.  Of 20 shapes 11 get the best, 6 more come within 16 %, the last are 24 and 36 % off.
  const long long each = (static_cast<long long>(T) * G + a.n_seq - 1) / a.n_seq, blocks = a.n_seq * ((each + kTfRows - 1) / kTfRows) * a.Hkv;
  long long keys = static_cast<long long>(a.max_blocks) * a.page_size / kTfKeys + 1;
  if (a.window != 0) keys = min(keys, llabs(static_cast<long long>(a.window)) / kTfKeys + 4);
  int cluster = kTfCluster;
  while (cluster > 1 && (blocks * cluster > 4ll * sms || cluster > keys || (blocks * cluster > 2ll * sms && 2 * cluster > keys))) cluster /= 2;
  if (tiles * cluster > 0x7fffffffll) return PMM_ERR_BAD_ARGUMENT;
  const size_t smem = tf_smem(a.Dh, sizeof(S));
  auto kern = a.window_step ? tree_rows_kernel<S, ACC, true> : tree_rows_kernel<S, ACC, false>;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));  // (of the current device: at every call)
  if (e != cudaSuccess) return static_cast<int>(e);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(tiles * cluster), a.Hkv);
  cfg.blockDim = dim3(kTfThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attrs[2]{};
  attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[0].val.programmaticStreamSerializationAllowed = 1;
  attrs[1].id = cudaLaunchAttributeClusterDimension;
  attrs[1].val.clusterDim.x = cluster;
  attrs[1].val.clusterDim.y = 1;
  attrs[1].val.clusterDim.z = 1;
  cfg.attrs = attrs;
  cfg.numAttrs = 2;
  cudaLaunchKernelEx(&cfg, kern, a, T, cluster);
  return launch_status();
}

}  // namespace pmm

// q [T, Hq*Dh], k, v [T, Hkv*Dh] with row strides in elements, rows on 16-byte boundaries; pool [pages, 2, page_size, Hkv*Dh]; out [T,
// Hq*Dh].  Rows behind the last request (cu[n_seq] and further) are left as they are.
PMM_EXPORT int pmm_tree_attention(const void* q, long long ldq, const void* k, long long ldk, const void* v, long long ldv, const void* pool, int pages,
                                  const int* block_table, int max_blocks, const int* held, const int* cu, const int* positions, const void* mask,
                                  int words, const float* sink, void* out, float scale, int window, int window_step, int page_size, int n_seq, int T,
                                  int Hq, int Hkv, int Dh, int dtype, int sms, cudaStream_t stream) {
  if (T <= 0 || n_seq <= 0) return 0;
  if (Dh <= 0 || Dh % 16 || Dh > 512 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || Hq > 65535 || page_size <= 0 || sms < 1 || max_blocks <= 0 || pages <= 0 || !(scale > 0.f) ||
      (window != 0 && !positions) || (mask && words < 1))
    return PMM_ERR_BAD_ARGUMENT;
  if (pmm::tree_attention_overlap(q, ldq, k, ldk, v, ldv, pool, pages, out, page_size, T, Hq, Hkv, Dh, dtype == 0 ? 4 : 2)) return PMM_ERR_OVERLAP;
  PMM_DISPATCH_DTYPE(dtype, S, {
    pmm::TreeAttnArgs<S> a{static_cast<const S*>(q), ldq, static_cast<const S*>(k), ldk, static_cast<const S*>(v), ldv, static_cast<const S*>(pool),
                           block_table, max_blocks, pages, held, cu, positions, static_cast<const unsigned long long*>(mask), words, sink,
                           static_cast<S*>(out), scale, window, window != 0 && window_step, page_size, n_seq, Hq, Hkv, Dh};
    if (Dh <= 64) return pmm::launch_tree_rows<S, 2>(a, T, sms, stream);
    if (Dh <= 128) return pmm::launch_tree_rows<S, 4>(a, T, sms, stream);
    if (Dh <= 256) return pmm::launch_tree_rows<S, 8>(a, T, sms, stream);
    pmm::launch_pdl(pmm::tree_attention_kernel<S, 16>, dim3(T, Hq), dim3(pmm::kTaWarps * 32), static_cast<size_t>(pmm::kTaWarps) * Dh * sizeof(float), stream, a, T);
  });
  return pmm::launch_status();
}
