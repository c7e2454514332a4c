// What the two launchers of the attention of drafted trees check alike.
#pragma once
#include "common.cuh"

namespace pmm {

// Whether results would be written where other blocks still read: in k, v or the pool, or in a part of q.  Into q itself they may go, row on
// row: whoever writes a row's result is the last to read its query, and parts of units that shares cut are merged by a later launch.
inline bool tree_attention_overlap(const void* q, long long ldq, const void* k, long long ldk, const void* v, long long ldv, const void* pool,
                                   long long pages, const void* out, int page_size, int T, int Hq, int Hkv, int Dh, int elem) {
  const long long q_row = static_cast<long long>(Hq) * Dh * elem, kv_row = static_cast<long long>(Hkv) * Dh * elem;
  const bool in_place = out == q && (T == 1 || ldq * elem == q_row);
  return (!in_place && rows_overlap(q, T, ldq * elem, q_row, out, T * q_row)) || rows_overlap(k, T, ldk * elem, kv_row, out, T * q_row) ||
         rows_overlap(v, T, ldv * elem, kv_row, out, T * q_row) || overlap(pool, pages * 2 * page_size * kv_row, out, T * q_row);
}

}  // namespace pmm
