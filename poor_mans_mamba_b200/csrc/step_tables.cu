// What surrounds a step of drafted tokens on the cache's side: block tables and the tokens' places built on the device from the
// requests' lengths, and the kept tokens' keys and values moved into the pages.
//
// step_tables, request s with held[s] cached tokens, new[s] tokens in this step and blocks[s] pages of its own:
//   after = max(blocks, ceil((held + new) / P)),  table[s, blocks .. after) = the next free pages, in the requests' order,
//   cu = running sums of new,  token i: position held + depth(i), slot = table[s, (held + i) / P] * P + (held + i) % P,
//   mask bit j = token j of the request is i or one of its ancestors (parents lie in front of their children).
// Nothing but latency bounds it: a block per request adds up the lengths of the requests in front of it (all loads of a thread
// go out together; 512 requests are two loads a thread and length) instead of a launch of its own for the sums.
//
// keep_accepted: rows[l, plane, cu[s] + path[s, j]] -> pool[l, slot / P, plane, slot % P], slot = slots[cu[s] + j], j < count[s].
// A copy: a block per (some layers and planes, request), a warp a row, up to eight pieces of a lane asked for before the first is stored.
//
// What these kernels write, later launches read ahead of their wait (sequence bounds, tables, cached keys): neither lets the
// launch behind it begin early, and both wait for their stores (pdl_arrived).
#include "common.cuh"

namespace pmm {

constexpr int kTablesThreads = 256;
constexpr int kTablesNodes = 1024;  // parents of a request kept in shared memory

struct StepTablesArgs {
  const int* held;
  const int* fresh;       // new tokens
  const int* blocks;
  int* table;             // [n, width]
  int width;
  const int* free_pages;
  int n_free, n, page_size, spare;
  int* cu;
  int* seq_of;
  int* positions;
  int* slots;
  int cap;                // tokens that the three have room for
  int* blocks_out;
  int* taken;
  const int* parents;     // [cap] or nullptr: chains
  unsigned long long* masks;
  int words;
};

__device__ __forceinline__ int saturated(long long x) { return static_cast<int>(min(x, 0x7fffffffll)); }

__device__ __forceinline__ int blocks_after(int held, int fresh, int blocks, int page_size) {
  return max(blocks, saturated((static_cast<long long>(held) + fresh + page_size - 1) / page_size));
}

__global__ void __launch_bounds__(kTablesThreads) step_tables_kernel(const StepTablesArgs a) {
  __shared__ long long s_sum[2][kTablesThreads / 32];
  __shared__ int s_up[kTablesNodes];
  pdl_wait();
  const int s = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int held = max(a.held[s], 0), fresh = max(a.fresh[s], 0), blocks = max(a.blocks[s], 0);
  // of the requests in front of this one (in 64 bits: lengths that fit no step must not come out as places in front of the tables)
  long long tokens = 0, pages = 0;
  for (int i = tid; i < s; i += kTablesThreads) {
    const int f = max(a.fresh[i], 0), b = max(a.blocks[i], 0);
    tokens += f;
    pages += blocks_after(max(a.held[i], 0), f, b, a.page_size) - b;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    tokens += __shfl_xor_sync(0xffffffffu, tokens, o);
    pages += __shfl_xor_sync(0xffffffffu, pages, o);
  }
  if (lane == 0) {
    s_sum[0][warp] = tokens;
    s_sum[1][warp] = pages;
  }
  __syncthreads();
  long long first = 0, g0 = 0;
#pragma unroll
  for (int w = 0; w < kTablesThreads / 32; ++w) {
    first += s_sum[0][w];
    g0 += s_sum[1][w];
  }
  const int after = blocks_after(held, fresh, blocks, a.page_size);
  const int t0 = saturated(first);
  if (tid == 0) {
    a.cu[s] = t0;
    a.blocks_out[s] = after;
    if (s == a.n - 1) {
      a.cu[a.n] = saturated(first + fresh);
      a.taken[0] = saturated(g0 + after - blocks);
    }
  }
  int* row = a.table + static_cast<size_t>(s) * a.width;
  // block b's page: one of the request's own, or the next free one
  auto page_of = [&](unsigned b) {
    if (b >= static_cast<unsigned>(a.width)) return a.spare;
    if (b < static_cast<unsigned>(blocks)) return row[b];
    const long long i = g0 + b - blocks;
    return i < a.n_free ? a.free_pages[i] : a.spare;
  };
  for (int b = min(blocks, a.width) + tid; b < a.width; b += kTablesThreads) row[b] = b < after ? page_of(b) : a.spare;

  const int n = min(fresh, a.cap - t0);  // (t0 <= cap unless the lengths do not fit the step)
  const bool cached = n <= kTablesNodes;
  if (a.parents != nullptr && cached) {
    for (int i = tid; i < n; i += kTablesThreads) s_up[i] = a.parents[t0 + i];
    __syncthreads();
  }
  for (int i = tid; i < n; i += kTablesThreads) {
    const int t = t0 + i;
    const unsigned pos = static_cast<unsigned>(held) + i, size = a.page_size;
    const int page = page_of(pos / size);
    const long long slot = static_cast<long long>(page) * a.page_size + pos % size;
    a.seq_of[t] = s;
    a.slots[t] = page < 0 || page == a.spare || slot > 0x7fffffffll ? -1 : static_cast<int>(slot);
    int depth = i;
    if (a.parents != nullptr) {
      depth = 0;
      unsigned long long bits[4] = {0ull, 0ull, 0ull, 0ull};
      for (int j = i;;) {
        if (j < 64 * a.words) {
#pragma unroll
          for (int w = 0; w < 4; ++w)
            if (j >> 6 == w) bits[w] |= 1ull << (j & 63);
        }
        const int up = cached ? s_up[j] : a.parents[t0 + j];
        if (up < 0 || up >= j) break;  // (a parent lies in front of its child: anything else is a root)
        j = up;
        ++depth;
      }
#pragma unroll
      for (int w = 0; w < 4; ++w)
        if (w < a.words) a.masks[static_cast<size_t>(t) * a.words + w] = bits[w];
    }
    a.positions[t] = saturated(static_cast<long long>(held) + depth);
  }
  pdl_arrived();
}

constexpr int kKeepThreads = 256;
constexpr int kKeepLoads = 4;   // pieces of a row that a lane has in flight
constexpr int kKeepPlanes = 4;  // layers and planes of a block where there are many
constexpr int kKeepResident = 4 * 148;  // blocks on the device at once (64 registers a thread)

// V: the piece that a thread copies at a time (16 bytes where rows begin on such boundaries).
template <typename V>
__global__ void __launch_bounds__(kKeepThreads, kKeepResident / 148)
    keep_accepted_kernel(const V* rows, long long ld_layer, long long ld_plane, long long ld_row, int n_rows, V* pool, long long pages,
                         int layers, int planes, int per_block, int page_size, int width, const int* slots, const int* cu, const int* path,
                         int path_width, const int* count) {
  pdl_wait();
  const int s = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t0 = max(cu[s], 0), t1 = min(max(cu[s + 1], 0), n_rows);  // (no bound leads out of the rows)
  const int kept = min(min(count[s], path_width), t1 - t0);
  if (kept <= 0) return;
  const int lp0 = blockIdx.x * per_block, n_lp = min(per_block, layers * planes - lp0);
  const long long n_slots = pages * page_size;
  constexpr int kWarps = kKeepThreads / 32;
  struct Row {
    const V* src;
    V* dst;
  };
  auto row = [&](int i) {  // row i of the block's: kept token i % kept of layer and plane lp0 + i / kept (none: no source)
    Row r{nullptr, nullptr};
    if (i >= kept * n_lp) return r;
    const int lp = lp0 + i / kept, j = i % kept, layer = lp / planes, plane = lp - layer * planes;
    const int node = path[static_cast<size_t>(s) * path_width + j], slot = slots[t0 + j];
    if (node < 0 || t0 + node >= t1 || slot < 0 || slot >= n_slots) return r;
    r.src = rows + layer * ld_layer + plane * ld_plane + static_cast<long long>(t0 + node) * ld_row;
    r.dst = pool + ((static_cast<long long>(layer) * pages + slot / page_size) * planes + plane) * page_size * width +
            static_cast<long long>(slot % page_size) * width;
    return r;
  };
  for (int i = warp; i < kept * n_lp; i += 2 * kWarps) {  // two rows at a time
    const Row r[2] = {row(i), row(i + kWarps)};
    for (int base = lane; base < width; base += 32 * kKeepLoads) {
      V v[2][kKeepLoads];
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int u = 0; u < kKeepLoads; ++u)
          if (r[k].src != nullptr && base + 32 * u < width) v[k][u] = r[k].src[base + 32 * u];
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int u = 0; u < kKeepLoads; ++u)
          if (r[k].src != nullptr && base + 32 * u < width) r[k].dst[base + 32 * u] = v[k][u];
    }
  }
  pdl_arrived();
}

}  // namespace pmm

// parents (with masks [cap, words], 1 to 4 words) or neither; table [n, width] and the lengths [n] contiguous.
PMM_EXPORT int pmm_step_tables(const int* held, const int* fresh, const int* blocks, int* table, int width, const int* free_pages, int n_free,
                               int n, int page_size, int spare, int* cu, int* seq_of, int* positions, int* slots, int cap, int* blocks_out,
                               int* taken, const int* parents, void* masks, int words, cudaStream_t stream) {
  if (n <= 0) return 0;
  if (width <= 0 || n_free < 0 || page_size <= 0 || spare < 0 || cap < 0 || (static_cast<long long>(spare) + 1) * page_size > 0x7fffffffll ||
      (parents == nullptr) != (masks == nullptr) || (parents && (words < 1 || words > 4)))
    return PMM_ERR_BAD_ARGUMENT;
  // Every request reads the lengths of those in front of it, and its own parents, while others write.
  const pmm::Extent written[] = {{cu, 4ll * (n + 1)}, {blocks_out, 4ll * n}, {taken, 4}, {table, 4ll * n * width}, {seq_of, 4ll * cap}, {positions, 4ll * cap},
                          {slots, 4ll * cap}, {masks, 8ll * cap * words}};
  const pmm::Extent read[] = {{held, 4ll * n}, {fresh, 4ll * n}, {blocks, 4ll * n}, {parents, 4ll * cap}};
  if (pmm::overlap(written, read)) return PMM_ERR_OVERLAP;
  for (int i = 0; i < 4; ++i)
    if (pmm::overlap(written[i].at, written[i].bytes, free_pages, 4ll * n_free)) return PMM_ERR_OVERLAP;
  pmm::StepTablesArgs a{held, fresh, blocks, table, width, free_pages, n_free, n, page_size, spare, cu, seq_of, positions, slots, cap, blocks_out,
                        taken, parents, static_cast<unsigned long long*>(masks), words};
  pmm::launch_pdl(pmm::step_tables_kernel, dim3(n), dim3(pmm::kTablesThreads), 0, stream, a);
  return pmm::launch_status();
}

// rows: strides in elements of `item` bytes; pool [layers, pages, planes, page_size, width] contiguous.
PMM_EXPORT int pmm_keep_accepted(const void* rows, long long ld_layer, long long ld_plane, long long ld_row, int n_rows, void* pool, int layers,
                                 long long pages, int planes, int page_size, int width, int item, const int* slots, const int* cu,
                                 const int* path, int path_width, const int* count, int n, cudaStream_t stream) {
  if (n <= 0 || layers <= 0 || planes <= 0) return 0;
  if (pages <= 0 || page_size <= 0 || width <= 0 || path_width <= 0 || n_rows < 0 || n > 65535 || (item != 2 && item != 4) ||
      static_cast<long long>(layers) * planes > 0x7fffffffll)
    return PMM_ERR_BAD_ARGUMENT;
  const long long pool_bytes = static_cast<long long>(layers) * pages * planes * page_size * width * item;
  for (int l = 0; l < layers; ++l)
    for (int p = 0; p < planes; ++p)
      if (pmm::rows_overlap(static_cast<const char*>(rows) + (l * ld_layer + p * ld_plane) * item, n_rows, ld_row * item,
                            static_cast<long long>(width) * item, pool, pool_bytes))
        return PMM_ERR_OVERLAP;
  // the widest piece that every row begins on
  const long long all = reinterpret_cast<uintptr_t>(rows) | reinterpret_cast<uintptr_t>(pool) | (ld_layer * item) | (ld_plane * item) |
                        (ld_row * item) | (static_cast<long long>(width) * item);
  // One plane a block while all blocks are on the device at once, two while half as many are, else four: a block that comes later than the
  // first ones waits for its three dependent reads once more.  5 of 8 tokens kept, us with one, two and four planes a block:
  //   planes x requests  576: 3.6  3.7  3.9    640: 5.2  4.0  4.8    896: 5.8  4.5  5.2 (rows of 1,024);   1,024: 5.0  3.9  4.3
  //   1,536: 6.9  5.9  4.9 (of 512);   2,048: 12.9  11.0  10.4    4,096: 22.5  19.2  18.7    8,192: 41.4  33.5  32.9 (of 1,024)
  const long long blocks = static_cast<long long>(layers) * planes * n;
  const int per_block = blocks <= pmm::kKeepResident ? 1 : blocks <= 2 * pmm::kKeepResident ? 2 : pmm::kKeepPlanes;
  const dim3 grid((layers * planes + per_block - 1) / per_block, n);
  auto go = [&](auto zero) {
    using V = decltype(zero);
    const int per = static_cast<int>(sizeof(V)) / item;
    pmm::launch_pdl(pmm::keep_accepted_kernel<V>, grid, dim3(pmm::kKeepThreads), 0, stream, static_cast<const V*>(rows), ld_layer / per,
                    ld_plane / per, ld_row / per, n_rows, static_cast<V*>(pool), pages, layers, planes, per_block, page_size, width / per, slots, cu, path, path_width,
                    count);
    return pmm::launch_status();
  };
  if (all % 16 == 0) return go(uint4{});
  if (all % 4 == 0) return go(0u);
  return go(static_cast<unsigned short>(0));
}
