// The requests' page tables on the device, and a step's maps built from them.
//
// Every request slot has a row of a table [slots, width]: the ids of its pages, in the order of its tokens.  The host sends
// only the cells that changed (pages taken since the last step); a step's block table, positions and slot map are made here
// from the requests' lengths:
//
//   start_r        = max(kv_len_r - count_r, 0)
//   q_start_r      = sum of counts of the entries before r
//   positions_n    = start_e + (n - q_start_e)                    for the tokens n of entry e
//   block_table_rc = tables[slots_r][c]  if c page_size < kv_len_r, else -1
//   slot_map_n     = block_table[e][p / page_size] page_size + p % page_size, or -1 where there is no page
//
// Nothing but copies of a few bytes per token and column: what bounds it is the launch (64 entries of 2,048 columns, the cells set and
// the maps made: 3.5 us).
#include "common.cuh"
#include "slots.h"

namespace b200 {

// tables[rows[i]][columns[i]] = pages[i].  A cell outside the table is left alone.
__global__ void page_table_set_kernel(int* __restrict__ tables, int table_rows, int width, const int* __restrict__ rows,
                                      const int* __restrict__ columns, const int* __restrict__ pages, int n) {
  pdl_trigger();
  pdl_wait();
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n) return;
  const int row = rows[i], column = columns[i];
  if (row < 0 || row >= table_rows || column < 0 || column >= width) return;
  tables[static_cast<size_t>(row) * width + column] = pages[i];
}

struct StepMapsArgs {
  const int* tables;
  const int* slots;
  const int* kv_len;
  const int* counts;
  int* block_table;
  int* q_start;        // the rest may be null: not wanted
  int* positions;
  int* token_entry;
  long long* slot_map;
  int table_rows, width, out_width, entries, page_size, num_tokens;
};

constexpr int kMapThreads = 256;
constexpr int kMapShare = 4 * kMapThreads;     // columns, and tokens, of an entry that one CTA takes at a time

// out[c] = row[c] for the columns below `held`, -1 behind them; VEC: four columns to a 16-byte access.
template <bool VEC>
__device__ __forceinline__ void copy_row(const int* row, int held, int* out, int out_width, int thread, int threads) {
  for (int c = thread * 4; c < out_width; c += threads * 4) {
    if (VEC) {
      int4 v = c < held ? *reinterpret_cast<const int4*>(row + c) : make_int4(-1, -1, -1, -1);
      if (c + 1 >= held) v.y = -1;
      if (c + 2 >= held) v.z = -1;
      if (c + 3 >= held) v.w = -1;
      *reinterpret_cast<int4*>(out + c) = v;
    } else {
      for (int i = c; i < min(c + 4, out_width); ++i) out[i] = i < held ? row[i] : -1;
    }
  }
}

// One CTA per (entry, share of its columns and tokens).  The tokens before an entry are counted by every CTA itself (a step
// has at most some hundred entries), so no CTA waits for another.
template <bool VEC>
__global__ void __launch_bounds__(kMapThreads) step_maps_kernel(const __grid_constant__ StepMapsArgs a) {
  __shared__ int warp_sums[kMapThreads / 32];
  pdl_trigger();
  pdl_wait();
  const int r = blockIdx.x, t = threadIdx.x;
  const int slot = a.slots[r], length = max(a.kv_len[r], 0), page_size = a.page_size;
  const bool known = slot >= 0 && slot < a.table_rows;
  const int* row = a.tables + static_cast<size_t>(known ? slot : 0) * a.width;
  const int held = known && length > 0 ? min((length - 1) / page_size + 1, a.width) : 0;      // columns that hold a page
  copy_row<VEC>(row, held, a.block_table + static_cast<size_t>(r) * a.out_width, a.out_width, blockIdx.y * kMapThreads + t, gridDim.y * kMapThreads);
  if (a.q_start == nullptr && a.positions == nullptr && a.token_entry == nullptr && a.slot_map == nullptr) return;
  int before = 0;
  for (int i = t; i < r; i += kMapThreads) before += max(a.counts[i], 0);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
  if ((t & 31) == 0) warp_sums[t >> 5] = before;
  __syncthreads();
  before = 0;
#pragma unroll
  for (int w = 0; w < kMapThreads / 32; ++w) before += warp_sums[w];
  const int count = max(a.counts[r], 0), start = max(length - count, 0);
  if (a.q_start != nullptr && blockIdx.y == 0 && t == 0) {
    a.q_start[r] = before;
    if (r == a.entries - 1) a.q_start[r + 1] = before + count;
  }
  for (int i = blockIdx.y * kMapThreads + t; i < count; i += gridDim.y * kMapThreads) {
    const int n = before + i;
    if (static_cast<unsigned>(n) >= static_cast<unsigned>(a.num_tokens)) break;
    const int position = start + i, column = position / page_size;
    if (a.positions != nullptr) a.positions[n] = position;
    if (a.token_entry != nullptr) a.token_entry[n] = r;
    if (a.slot_map != nullptr) {
      const int page = column < held ? row[column] : -1;
      a.slot_map[n] = page < 0 ? -1 : static_cast<long long>(page) * page_size + (position - column * page_size);
    }
  }
}

// The start of a step of single decoded tokens: what b200_slot_load does (slots.cu), and the block table's row of each entry, one
// CTA each; the record is read before it is advanced, and by nobody else.
struct SlotMapsArgs {
  int* records;
  const int* slots;
  int* token_ids;
  int* positions;
  int* kv_len;
  const int* tables;
  int* block_table;
  int records_count, table_rows, width, out_width, page_size;
};

template <bool VEC>
__global__ void __launch_bounds__(kMapThreads) slot_load_maps_kernel(const __grid_constant__ SlotMapsArgs a) {
  __shared__ int shared_length;
  pdl_trigger();
  pdl_wait();
  const int r = blockIdx.x, t = threadIdx.x, slot = a.slots[r];
  if (t == 0) {
    int* rec = a.records + static_cast<size_t>(slot) * kSlotWords;
    const bool live = slot >= 0 && slot < a.records_count && rec[kSlotLive] != 0;
    const int pos = live ? rec[kSlotPosition] : 0, token = live ? rec[kSlotLastToken] : 0;
    a.token_ids[r] = token < 0 ? 0 : token;      // a refused draw (-1: non-finite logits) is reported by the host; never index with it
    a.positions[r] = pos;
    a.kv_len[r] = live ? pos + 1 : 0;
    if (live) rec[kSlotPosition] = pos + 1;
    shared_length = live ? pos + 1 : 0;
  }
  __syncthreads();
  const int length = max(shared_length, 0);
  const bool known = slot >= 0 && slot < a.table_rows;
  const int held = known && length > 0 ? min((length - 1) / a.page_size + 1, a.width) : 0;
  copy_row<VEC>(a.tables + static_cast<size_t>(known ? slot : 0) * a.width, held, a.block_table + static_cast<size_t>(r) * a.out_width,
                a.out_width, t, kMapThreads);
}

bool vector_rows(const int* tables, int width, const int* block_table, int out_width) {
  return width % 4 == 0 && out_width % 4 == 0 && reinterpret_cast<uintptr_t>(tables) % 16 == 0 && reinterpret_cast<uintptr_t>(block_table) % 16 == 0;
}

}  // namespace b200

using namespace b200;

extern "C" int b200_page_table_set(int* tables, int table_rows, int width, const int* rows, const int* columns, const int* pages,
                                   int n, cudaStream_t stream) {
  if (n <= 0) return 0;
  if (table_rows <= 0 || width <= 0) return B200_ERR_BAD_SIZE;
  const int threads = 128;
  launch(page_table_set_kernel, dim3((n + threads - 1) / threads), dim3(threads), 0, stream, tables, table_rows, width, rows, columns,
         pages, n);
  return launch_status();
}

extern "C" int b200_step_maps(const int* tables, int table_rows, int width, const int* slots, const int* kv_len, const int* counts,
                              int* block_table, int out_width, int* q_start, int* positions, int* token_entry, long long* slot_map,
                              int entries, int page_size, int num_tokens, cudaStream_t stream) {
  if (entries <= 0) return 0;
  if (table_rows <= 0 || width <= 0 || out_width <= 0 || page_size <= 0 || num_tokens < 0) return B200_ERR_BAD_SIZE;
  StepMapsArgs a{tables, slots, kv_len, counts, block_table, q_start, positions, token_entry, slot_map,
                 table_rows, width, out_width, entries, page_size, num_tokens};
  const bool vec = vector_rows(tables, width, block_table, out_width);
  // as many shares as the wider of a row's columns and a mean entry's tokens asks for
  const int tokens = (num_tokens + entries - 1) / entries;
  int shares = ((out_width > tokens ? out_width : tokens) + kMapShare - 1) / kMapShare;
  if (shares > 64) shares = 64;
  launch(vec ? step_maps_kernel<true> : step_maps_kernel<false>, dim3(entries, shares), dim3(kMapThreads), 0, stream, a);
  return launch_status();
}

extern "C" int b200_slot_load_maps(int* records, int records_count, const int* slots, int* token_ids, int* positions, int* kv_len,
                                   const int* tables, int table_rows, int width, int* block_table, int out_width, int entries,
                                   int page_size, cudaStream_t stream) {
  if (entries <= 0) return 0;
  if (records_count <= 0 || table_rows <= 0 || width <= 0 || out_width <= 0 || page_size <= 0) return B200_ERR_BAD_SIZE;
  SlotMapsArgs a{records, slots, token_ids, positions, kv_len, tables, block_table, records_count, table_rows, width, out_width, page_size};
  launch(vector_rows(tables, width, block_table, out_width) ? slot_load_maps_kernel<true> : slot_load_maps_kernel<false>, dim3(entries),
         dim3(kMapThreads), 0, stream, a);
  return launch_status();
}
