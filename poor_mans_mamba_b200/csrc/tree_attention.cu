// Attention of drafted tokens over a paged cache: token i of request s sees the request's held[s] cached keys (the last
// `window` positions up to its own, where there is a window) and, among the request's own tokens of this step, those whose
// bits its mask holds (without masks: those in front of it, and itself).
//   sc[j] = (q.K[j]) * scale;  p = exp(sc - max);  o = sum p V / sum p,   0 for a row that sees no key
// The step's own keys and values lie densely in k and v: the cache takes only those that are kept in the end.
//
// This kernel: float arithmetic on the CUDA cores, any storage type and head size.  A block per (token, query head); its eight
// warps share the keys in pieces of 32 (a key per lane for the scores, a slice of the head per lane for the values) and merge
// their maxima, sums and results at the end.  The keys of a group's query heads are read once per head, from L2.
#include "common.cuh"
#include <math_constants.h>

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
  int window, page_size, n_seq, Hq, Hkv, Dh;
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

template <typename S, int ACC>
__global__ void __launch_bounds__(kTaWarps * 32) tree_attention_kernel(const TreeAttnArgs<S> a) {
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
  const int t0 = a.cu[seq], n_new = a.cu[seq + 1] - t0, held = max(0, static_cast<int>(min(static_cast<long long>(a.held[seq]), static_cast<long long>(a.max_blocks) * a.page_size)));
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
      const bool valid = j < end && (part == 0 || (mask ? ta_sees(mask, a.words, j) : j <= t - t0));
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
      // values of kKeys keys at a time, so that as many rows travel together (one behind the other a row costs an L2 latency: 32 us
      // where 4 requests with 12 tokens and 8 heads see 300 keys, together 21); of keys that are not seen they may be anything
      constexpr int kKeys = ACC <= 4 ? 8 : 32 / ACC;
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
  if (a.sink && warp == 0) {  // a score without key or value that counts once
    const float m_new = fmaxf(m, a.sink[hq]);
    const float corr = expf(m - m_new);
    l = l * corr + expf(a.sink[hq] - m_new);
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

}  // namespace pmm

// q [T, Hq*Dh], k, v [T, Hkv*Dh] with row strides in elements, rows on 16-byte boundaries; pool [pages, 2, page_size, Hkv*Dh]; out [T,
// Hq*Dh].  Rows behind the last request (cu[n_seq] and further) are left as they are.
PMM_EXPORT int pmm_tree_attention(const void* q, long long ldq, const void* k, long long ldk, const void* v, long long ldv, const void* pool, int pages,
                                  const int* block_table, int max_blocks, const int* held, const int* cu, const int* positions, const void* mask,
                                  int words, const float* sink, void* out, float scale, int window, int page_size, int n_seq, int T, int Hq,
                                  int Hkv, int Dh, int dtype, cudaStream_t stream) {
  if (T <= 0 || n_seq <= 0) return 0;
  if (Dh <= 0 || Dh % 16 || Dh > 512 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || Hq > 65535 || page_size <= 0 || max_blocks <= 0 || pages <= 0 || !(scale > 0.f) ||
      (window != 0 && !positions) || (mask && words < 1))
    return PMM_ERR_BAD_ARGUMENT;
  PMM_DISPATCH_DTYPE(dtype, S, {
    pmm::TreeAttnArgs<S> a{static_cast<const S*>(q), ldq, static_cast<const S*>(k), ldk, static_cast<const S*>(v), ldv, static_cast<const S*>(pool),
                           block_table, max_blocks, pages, held, cu, positions, static_cast<const unsigned long long*>(mask), words, sink,
                           static_cast<S*>(out), scale, window, page_size, n_seq, Hq, Hkv, Dh};
    auto kern = Dh <= 64 ? pmm::tree_attention_kernel<S, 2> : Dh <= 128 ? pmm::tree_attention_kernel<S, 4>
              : Dh <= 256 ? pmm::tree_attention_kernel<S, 8> : pmm::tree_attention_kernel<S, 16>;
    pmm::launch_pdl(kern, dim3(T, Hq), dim3(pmm::kTaWarps * 32), static_cast<size_t>(pmm::kTaWarps) * Dh * sizeof(float), stream, a);
  });
  return pmm::launch_status();
}
