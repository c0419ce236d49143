// Attention of every query row over the keys of the pages chosen for it and its kv head:
//
//   out_h = sum_k exp(scale q_h.k) v_k / sum_k exp(scale q_h.k)
//
// over the keys k of the listed pages at positions up to the row's own.  Each page of keys and values is read once for all heads
// of the group; what bounds it is that reading (from HBM for single tokens, from L2 for the rows of a prompt).
//
// The pages of a list are dealt out to the `parts` CTAs of a cluster in turn, the keys of a CTA's pages to its warps; every warp
// (or team of lanes) keeps a running maximum, a sum and the weighted values, which are joined over shared memory, the parts over
// the cluster's.  Nothing is kept between launches.
#include "mma.cuh"
#include "sparse_pages.cuh"

namespace b200 {

struct AttendArgs {
  const void* q;
  const void* keys;
  const void* values;
  const int* chosen;
  const int* positions;
  const int* token_entry;
  const int* block_table;
  void* out;
  int table_width, rows, entries, q_heads, kv_heads, page_size, num_pages, budget, parts;
  float scale_log2;       // scale / ln 2: weights are powers of two
};

constexpr int kPlaces = 512;       // pages of a list that a CTA looks up at a time
constexpr int kSumsRow = kDim + 1; // a row of weighted values in shared memory: what the lanes of a fragment write falls on 32 banks

struct Place {
  int page;     // page of the pool
  int last;     // last slot of it that the row sees; negative: none
};

struct Work {
  int row, head, slice, part;
};

// Rows follow one another head by head: the rows of a prompt that run at once then read the pages of one or two heads, which L2 holds
// (874 rows: 555 us instead of 587, and 570 on pages that are not in L2 yet, where it had been 650).
__device__ __forceinline__ Work work_of(const AttendArgs& a, int slices) {
  int x = blockIdx.x;
  Work w;
  w.part = x % a.parts;
  x /= a.parts;
  w.slice = x % slices;
  x /= slices;
  w.row = x % a.rows;
  w.head = x / a.rows;
  return w;
}

// Places from .. of this part's share of the row's list (page place * parts + part of it): how many there are; all threads.
__device__ __forceinline__ int look_up(const AttendArgs& a, const Work& w, int from, int entry, int position, Place* places, int threads) {
  const int share = (a.budget - w.part + a.parts - 1) / a.parts;
  const int count = min(share - from, kPlaces);
  const int* chosen = a.chosen + (static_cast<size_t>(w.row) * a.kv_heads + w.head) * a.budget;
  const int* table = a.block_table + static_cast<size_t>(entry) * a.table_width;
  for (int i = threadIdx.x; i < count; i += threads) {
    const int column = chosen[(from + i) * a.parts + w.part];
    Place place{0, -1};
    if (column >= 0 && column < a.table_width) {
      const int page = table[column];
      const long long last = position - static_cast<long long>(column) * a.page_size;
      if (page >= 0 && page < a.num_pages && last >= 0) place = Place{page, static_cast<int>(min(last, static_cast<long long>(a.page_size - 1)))};
    }
    places[i] = place;
  }
  return count;
}

// Joins what the warps of a CTA hold, then what the CTAs of a cluster hold, and writes the heads' rows: sums[w][h][c] are the
// warps' weighted values, top[w][h] and total[w][h] their maxima and sums.  All threads of all parts; the order of every sum is
// that of the warps and of the parts.
template <typename T, int WARPS, int H>
__device__ void join_and_write(const AttendArgs& a, const Work& w, float (*sums)[H][kSumsRow], float (*top)[H], float (*total)[H], int heads_here,
                               T* out) {
  __shared__ float joined_top[H], joined_total[H];
  constexpr int kThreads = WARPS * 32;
  const int t = threadIdx.x;
  __syncthreads();
  for (int i = t; i < heads_here * kDim; i += kThreads) {
    const int h = i / kDim, c = i % kDim;
    float m = top[0][h];
#pragma unroll
    for (int v = 1; v < WARPS; ++v) m = fmaxf(m, top[v][h]);
    float x = 0.f, l = 0.f;
#pragma unroll
    for (int v = 0; v < WARPS; ++v) {
      // a warp that has seen nothing counts nothing; a NaN stays one
      const float factor = top[v][h] == -CUDART_INF_F ? 0.f : exp2f(top[v][h] - m);
      x = fmaf(sums[v][h][c], factor, x);
      l = fmaf(total[v][h], factor, l);
    }
    if (a.parts == 1) {
      out[i] = from_float<T>(l == 0.f ? 0.f : x / l);
    } else {
      sums[0][h][c] = x;
      if (c == 0) joined_top[h] = m, joined_total[h] = l;
    }
  }
  if (a.parts == 1) return;
  __syncthreads();                      // the cluster's barriers want whole warps
  cluster_arrive();
  cluster_wait();                       // every part's sums are in its CTA's shared memory
  const uint32_t sums_at = shared_address(&sums[0][0][0]), top_at = shared_address(joined_top), total_at = shared_address(joined_total);
  for (int i = w.part * kThreads + t; i < heads_here * kDim; i += a.parts * kThreads) {
    const int h = i / kDim, at = h * kSumsRow + i % kDim;
    float m = -CUDART_INF_F;
    for (int p = 0; p < a.parts; ++p) m = fmaxf(m, load_in_cluster(in_cluster(top_at + h * 4, p)));
    float x = 0.f, l = 0.f;
    for (int p = 0; p < a.parts; ++p) {
      const float own = load_in_cluster(in_cluster(top_at + h * 4, p));
      const float factor = own == -CUDART_INF_F ? 0.f : exp2f(own - m);
      x = fmaf(load_in_cluster(in_cluster(sums_at + at * 4, p)), factor, x);
      l = fmaf(load_in_cluster(in_cluster(total_at + h * 4, p)), factor, l);
    }
    out[i] = from_float<T>(l == 0.f ? 0.f : x / l);
  }
  __syncthreads();
  cluster_leave();                      // nobody leaves while its sums are being read
}

// ------------------------------------------------------------------------------------------------- float32, CUDA cores
// A few lanes hold a key's row (RowLanes), each such team walks keys of its own.  Which keys a team takes, and the order of every
// sum, depend on the list alone: `parts` is chosen from the list's length, not from the batch.  What bounds it is the latency of the
// keys in flight (240 registers: queries, values and two keys a team; 4 warps of a multiprocessor's 64 for one row): 90 rows, 2 kv heads
// of 64, 384 keys 13 us; one row, 8 of 128, 2,048 keys 16 us, 21 from HBM; 64 rows of 64 heads over 8, 2,048 keys 666 us (1.6 TB/s); 874
// rows of 16 heads over 8, 2,048 keys 3.7 ms (all their 10,000 to 16,000 keys by the dense kernel: 4.4).
struct Streams {
  using R = RowLanes<float>;
  static constexpr int threads = 128;
  static constexpr int heads = R::values <= 16 ? 4 : (R::values <= 32 ? 2 : 1);     // query heads a CTA takes
  static constexpr int ahead = R::values <= 16 ? 2 : 1;                             // keys of a team in flight
};

__global__ void __launch_bounds__(Streams::threads) attend_streams_kernel(const __grid_constant__ AttendArgs a) {
  using R = RowLanes<float>;
  constexpr int H = Streams::heads, V = R::values, U = Streams::ahead, kWarps = Streams::threads / 32, kTeams = Streams::threads / R::lanes;
  __shared__ float sums[kWarps][H][kSumsRow];
  __shared__ float top[kWarps][H], total[kWarps][H];
  __shared__ Place places[kPlaces];
  pdl_trigger();
  pdl_wait();
  const int group = a.q_heads / a.kv_heads;
  const Work w = work_of(a, (group + H - 1) / H);
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, part = t % R::lanes, team = t / R::lanes;
  const int heads_here = min(H, group - w.slice * H);
  const int entry = a.token_entry[w.row], position = a.positions[w.row];
  const bool stands = position >= 0 && entry >= 0 && entry < a.entries;
  const size_t q_row = (static_cast<size_t>(w.row) * a.q_heads + w.head * group + w.slice * H) * kDim;
  float q[H][V], o[H][V], m[H], l[H];
#pragma unroll
  for (int h = 0; h < H; ++h) {
    m[h] = -CUDART_INF_F, l[h] = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) q[h][i] = o[h][i] = 0.f;
    if (h < heads_here) {
      const float4* row = reinterpret_cast<const float4*>(static_cast<const float*>(a.q) + q_row + h * kDim);
#pragma unroll
      for (int i = 0; i < R::per_lane; ++i) {
        const float4 v = row[part + i * R::lanes];
        q[h][4 * i] = v.x * a.scale_log2, q[h][4 * i + 1] = v.y * a.scale_log2, q[h][4 * i + 2] = v.z * a.scale_log2, q[h][4 * i + 3] = v.w * a.scale_log2;
      }
    }
  }
  const unsigned team_lanes = ((1u << R::lanes) - 1u) << (lane / R::lanes * R::lanes);
  for (int from = 0; stands && from * a.parts + w.part < a.budget; from += kPlaces) {
    __syncthreads();
    const int keys = look_up(a, w, from, entry, position, places, Streams::threads) * a.page_size;
    __syncthreads();
    for (int k = team; k < keys; k += U * kTeams) {
      float kf[U][V], vf[U][V];
      bool is[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = k + u * kTeams, place = i / a.page_size, slot = i - place * a.page_size;
        is[u] = i < keys && slot <= places[place].last;
        if (!is[u]) continue;
        const size_t at = ((static_cast<size_t>(places[place].page) * a.kv_heads + w.head) * a.page_size + slot) * (kDim / 4) + part;
        const float4* key = static_cast<const float4*>(a.keys) + at;
        const float4* value = static_cast<const float4*>(a.values) + at;
#pragma unroll
        for (int c = 0; c < R::per_lane; ++c) Vec<float>::unpack(key[c * R::lanes], kf[u] + 4 * c);
#pragma unroll
        for (int c = 0; c < R::per_lane; ++c) Vec<float>::unpack(value[c * R::lanes], vf[u] + 4 * c);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (!is[u]) continue;
#pragma unroll
        for (int h = 0; h < H; ++h) {
          float s = 0.f;
#pragma unroll
          for (int c = 0; c < V; ++c) s = fmaf(q[h][c], kf[u][c], s);
#pragma unroll
          for (int x = 1; x < R::lanes; x <<= 1) s += __shfl_xor_sync(team_lanes, s, x);
          const float most = fmaxf(m[h], s);
          const float keep = m[h] == most ? 1.f : exp2f(m[h] - most);
          const float p = s == -CUDART_INF_F ? 0.f : exp2f(s - most);
          m[h] = most;
          l[h] = l[h] * keep + p;
#pragma unroll
          for (int c = 0; c < V; ++c) o[h][c] = fmaf(p, vf[u][c], o[h][c] * keep);
        }
      }
    }
  }
  __syncwarp();
#pragma unroll
  for (int h = 0; h < H; ++h) {        // the warp's teams
    float most = m[h];
#pragma unroll
    for (int x = R::lanes; x < 32; x <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, x));
    const float factor = m[h] == -CUDART_INF_F ? 0.f : exp2f(m[h] - most);
    float sum = l[h] * factor;
#pragma unroll
    for (int x = R::lanes; x < 32; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
#pragma unroll
    for (int c = 0; c < V; ++c) {
      float v = o[h][c] * factor;
#pragma unroll
      for (int x = R::lanes; x < 32; x <<= 1) v += __shfl_xor_sync(0xffffffffu, v, x);
      if (lane < R::lanes) sums[warp][h][(part + c / 4 * R::lanes) * 4 + c % 4] = v;
    }
    if (lane == 0) top[warp][h] = most, total[warp][h] = sum;
  }
  join_and_write<float, kWarps, H>(a, w, sums, top, total, heads_here, static_cast<float*>(a.out) + q_row);
}

// --------------------------------------------------------------------------------------------- bfloat16, tensor cores
// S^T = K Q^T and O^T = V^T P^T with mma.m16n8k16, keys (and value columns) as the 16 rows, the group's query heads as the 8
// columns: a group has few heads, so this way round nothing of the 16 rows is padding.  Keys and values are loaded from global
// memory straight into registers, 16 bytes a lane: lane (g, t) takes channels 8 t .. 8 t + 7 of every 32 of the rows g and g + 8 of
// a tile of 16 keys.  The sum over channels does not mind their order, so these are the fragments of K where they lie.  Values
// (and the weights P^T, which come in the layout of the accumulator) are turned by movmatrix, 8x8 numbers across the warp.  No
// shared memory and no barrier in the loop.
//
// Weights are rounded to bfloat16 where they meet the values (one operand type to a product; a second product for what the rounding
// leaves would be half as much work again); their sum is taken before, in 32 bits.  The rounding errors, 2^-8 of a weight at most, average
// out over the keys: the outputs' error against 64 bits is 1.7e-3 to 1.8e-3 of their norm, 1.66e-3 being that of the outputs' own rounding.
//
// Eight neighbouring lanes load from two rows, which lie on the same banks of the L1 cache where a row is a multiple of 128 bytes;
// odd rows then take the blocks of 32 channels of each pair in the other order and exchange the registers afterwards.  (874 prompt
// rows, 8 kv heads, 2,048 keys each: the data stage of L1 was 91 % busy with values read by columns and both kinds on shared banks, and
// the kernel took 747 us; 555 now.)  64 requests of 64 heads over 8, 2,048 keys each: 539 MB in 88 us, 6.1 TB/s.  Rows of a prompt are
// bound by L1's data stage (66 % busy): every row reads its own 8 MB of pages.  Dense tiles over all keys of the same rows, 6.6 times as
// many, take 250 us.
__device__ __forceinline__ uint4 load_row_16(const __nv_bfloat16* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ uint2 load_row_8(const __nv_bfloat16* p) {
  uint2 v;
  asm volatile("ld.global.L1::no_allocate.v2.u32 {%0, %1}, [%2];\n" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(r) : "r"(v));
  return r;
}

// 2^x of a weight that is rounded to bfloat16 next: to 22 bits, results below 2^-126 as 0.
__device__ __forceinline__ float power_of_two(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(r) : "f"(x));
  return r;
}

constexpr int kRowRegs = kDim / 8;              // registers of a lane for its channels of one row: pairs
constexpr int kTiles = kDim / 16;                // tiles of 16 value columns
constexpr bool kSwapOdd = kDim % 64 == 0;       // rows of whole 128 bytes

// A lane's channels of one row: 8 t .. 8 t + 7 of every 32, 4 t .. 4 t + 3 of the last 16.  ALL: the row is one to read.
template <bool ALL> __device__ __forceinline__ void load_channels(uint32_t (&r)[kRowRegs], const __nv_bfloat16* row, int t, bool odd, bool is) {
#pragma unroll
  for (int b = 0; b < kDim / 32; ++b) {
    uint4 v = make_uint4(0, 0, 0, 0);
    if (ALL || is) v = load_row_16(row + 32 * (kSwapOdd && odd ? b ^ 1 : b) + 8 * t);
    r[4 * b] = v.x, r[4 * b + 1] = v.y, r[4 * b + 2] = v.z, r[4 * b + 3] = v.w;
  }
  if (kDim % 32) {
    uint2 v = make_uint2(0, 0);
    if (ALL || is) v = load_row_8(row + kDim / 32 * 32 + 4 * t);
    r[kRowRegs - 2] = v.x, r[kRowRegs - 1] = v.y;
  }
}
// Puts the blocks of an odd row into their places.
__device__ __forceinline__ void order_channels(uint32_t (&r)[kRowRegs], bool odd) {
  if constexpr (kSwapOdd) {
#pragma unroll
    for (int i = 0; i < kRowRegs / 2; ++i) {
      const int a = i / 4 * 8 + i % 4, b = a + 4;
      const uint32_t x = r[a], y = r[b];
      r[a] = odd ? y : x, r[b] = odd ? x : y;
    }
  }
}
// The column that row g (half 0) or g + 8 (half 1) of tile m of O^T stands for: registers 2 m and 2 m + 1 of a lane hold columns of
// which the transposition hands two neighbours to neighbouring rows.
__device__ __forceinline__ int column_of(int m, int half, int g) {
  if (kDim % 32 && m == kDim / 16 - 1) return 16 * m + 4 * (g >> 1) + 2 * half + (g & 1);
  return 32 * (m / 2) + 8 * (g >> 1) + 4 * (m % 2) + 2 * half + (g & 1);
}

// NT: tiles of eight query heads of a CTA.  WHOLE: pages are whole tiles of 16 keys, so that a tile is a run of rows.
template <int NT, int WARPS, bool WHOLE>
__global__ void __launch_bounds__(WARPS * 32, NT == 1 && kDim <= 128 ? 16 / WARPS : 1) attend_mma_kernel(const __grid_constant__ AttendArgs a) {
  constexpr int H = 8 * NT;
  __shared__ float sums[WARPS][H][kSumsRow];
  __shared__ float top[WARPS][H], total[WARPS][H];
  __shared__ Place places[kPlaces];
  pdl_trigger();
  pdl_wait();
  const int group = a.q_heads / a.kv_heads;
  const Work w = work_of(a, (group + H - 1) / H);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const bool odd = g & 1;
  const int heads_here = min(H, group - w.slice * H);
  const int entry = a.token_entry[w.row], position = a.positions[w.row];
  const bool stands = position >= 0 && entry >= 0 && entry < a.entries;
  const size_t q_row = (static_cast<size_t>(w.row) * a.q_heads + w.head * group + w.slice * H) * kDim;
  uint32_t q[NT][kRowRegs];
#pragma unroll
  for (int n = 0; n < NT; ++n) load_channels<false>(q[n], static_cast<const __nv_bfloat16*>(a.q) + q_row + (8 * n + g) * kDim, t, false, 8 * n + g < heads_here);
  float o[NT][kTiles][4], m[NT][2], l[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    m[n][0] = m[n][1] = -CUDART_INF_F, l[n][0] = l[n][1] = 0.f;
#pragma unroll
    for (int i = 0; i < kTiles; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
  }
  const __nv_bfloat16* keys = static_cast<const __nv_bfloat16*>(a.keys) + static_cast<size_t>(w.head) * a.page_size * kDim;
  const __nv_bfloat16* values = static_cast<const __nv_bfloat16*>(a.values) + static_cast<size_t>(w.head) * a.page_size * kDim;
  const size_t page_stride = static_cast<size_t>(a.kv_heads) * a.page_size * kDim;
  for (int from = 0; stands && from * a.parts + w.part < a.budget; from += kPlaces) {
    __syncthreads();
    const int count = look_up(a, w, from, entry, position, places, WARPS * 32);
    __syncthreads();
    const int per_place = a.page_size / 16;         // WHOLE: tiles of a page
    const int tiles = WHOLE ? count * per_place : (count * a.page_size + 15) / 16;
    for (int tile = warp; tile < tiles; tile += WARPS) {
      size_t at[2];        // where the lane's rows g and g + 8 lie
      bool is[2];
      if (WHOLE) {
        const int place = tile / per_place, slot = (tile - place * per_place) * 16;
        const Place here = places[place];
        const int last = here.last - slot;
        if (last < 0) continue;                      // the same for the whole warp
#pragma unroll
        for (int i = 0; i < 2; ++i) at[i] = here.page * page_stride + static_cast<size_t>(slot + g + 8 * i) * kDim, is[i] = g + 8 * i <= last;
      } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int k = tile * 16 + g + 8 * i, place = k / a.page_size, slot = k - place * a.page_size;
          const Place here = place < count ? places[place] : Place{0, -1};
          at[i] = here.page * page_stride + static_cast<size_t>(slot) * kDim, is[i] = slot <= here.last;
        }
      }
      uint32_t k0[kRowRegs], k1[kRowRegs], v0[kRowRegs], v1[kRowRegs];
      if (__all_sync(0xffffffffu, is[0] && is[1])) {        // most tiles: nothing to blank out
        load_channels<true>(k0, keys + at[0], t, odd, true);
        load_channels<true>(k1, keys + at[1], t, odd, true);
        load_channels<true>(v0, values + at[0], t, odd, true);
        load_channels<true>(v1, values + at[1], t, odd, true);
      } else {
        load_channels<false>(k0, keys + at[0], t, odd, is[0]);
        load_channels<false>(k1, keys + at[1], t, odd, is[1]);
        load_channels<false>(v0, values + at[0], t, odd, is[0]);
        load_channels<false>(v1, values + at[1], t, odd, is[1]);
      }
      order_channels(k0, odd);
      order_channels(k1, odd);
      uint32_t weights[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float s[2][4] = {};        // two sums, so that each product waits for the one before the last
#pragma unroll
        for (int i = 0; i < kRowRegs / 2; ++i) mma_bf16(s[i & 1], {k0[2 * i], k1[2 * i], k0[2 * i + 1], k1[2 * i + 1]}, q[n][2 * i], q[n][2 * i + 1]);
        float keep[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {                // heads 2 t and 2 t + 1; keys g and g + 8
          float x = is[0] ? (s[0][c] + s[1][c]) * a.scale_log2 : -CUDART_INF_F;
          float y = is[1] ? (s[0][2 + c] + s[1][2 + c]) * a.scale_log2 : -CUDART_INF_F;
          float most = fmaxf(x, y);
          most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 4));
          most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 8));
          most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 16));
          most = fmaxf(most, m[n][c]);
          const float base = most == -CUDART_INF_F ? 0.f : most;
          keep[c] = power_of_two(m[n][c] - base);
          m[n][c] = most;
          x = power_of_two(x - base), y = power_of_two(y - base);
          l[n][c] = l[n][c] * keep[c] + x + y;
          s[0][c] = x, s[0][2 + c] = y;
        }
        weights[n][0] = transpose_8x8(pack_bf16(s[0][0], s[0][1]));
        weights[n][1] = transpose_8x8(pack_bf16(s[0][2], s[0][3]));
        if (__any_sync(0xffffffffu, keep[0] != 1.f || keep[1] != 1.f)) {
#pragma unroll
          for (int i = 0; i < kTiles; ++i) o[n][i][0] *= keep[0], o[n][i][1] *= keep[1], o[n][i][2] *= keep[0], o[n][i][3] *= keep[1];
        }
      }
      order_channels(v0, odd);
      order_channels(v1, odd);
#pragma unroll
      for (int i = 0; i < kTiles; ++i) {
        const uint32_t turned[4] = {transpose_8x8(v0[2 * i]), transpose_8x8(v0[2 * i + 1]), transpose_8x8(v1[2 * i]), transpose_8x8(v1[2 * i + 1])};
#pragma unroll
        for (int n = 0; n < NT; ++n) mma_bf16(o[n][i], turned, weights[n][0], weights[n][1]);
      }
    }
  }
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int h = 8 * n + 2 * t + c;
      float sum = l[n][c];
      sum += __shfl_xor_sync(0xffffffffu, sum, 4);
      sum += __shfl_xor_sync(0xffffffffu, sum, 8);
      sum += __shfl_xor_sync(0xffffffffu, sum, 16);
      if (g == 0) top[warp][h] = m[n][c], total[warp][h] = sum;
#pragma unroll
      for (int i = 0; i < kTiles; ++i) sums[warp][h][column_of(i, 0, g)] = o[n][i][c], sums[warp][h][column_of(i, 1, g)] = o[n][i][2 + c];
    }
  }
  join_and_write<__nv_bfloat16, WARPS, H>(a, w, sums, top, total, heads_here, static_cast<__nv_bfloat16*>(a.out) + q_row);
}

template <typename Kernel> int launch_attend(Kernel kernel, const AttendArgs& a, int heads, int warps, cudaStream_t stream) {
  const long long slices = (a.q_heads / a.kv_heads + heads - 1) / heads;
  const long long ctas = static_cast<long long>(a.rows) * a.kv_heads * slices * a.parts;
  if (ctas > 0x7fffffffll) return B200_ERR_TOO_LARGE;
  launch_clusters(kernel, dim3(static_cast<unsigned>(ctas)), dim3(warps * 32), 0, a.parts, stream, a);
  return launch_status();
}

template <int NT, int WARPS> int launch_mma(const AttendArgs& a, cudaStream_t stream) {
  return a.page_size % 16 == 0 ? launch_attend(attend_mma_kernel<NT, WARPS, true>, a, 8 * NT, WARPS, stream)
                               : launch_attend(attend_mma_kernel<NT, WARPS, false>, a, 8 * NT, WARPS, stream);
}

}  // namespace b200

using namespace b200;

// parts: CTAs of a cluster that share out a list; wide: eight warps to a CTA where there is such a kernel (bfloat16, head sizes up to
// 128, up to eight heads a group).
extern "C" int b200_attend_chosen(const void* q, const void* keys, const void* values, const int* chosen, const int* positions,
                                  const int* token_entry, const int* block_table, int table_width, void* out, int rows, int entries,
                                  int q_heads, int kv_heads, int page_size, int num_pages, int budget, float scale, int parts, int wide, int dtype,
                                  cudaStream_t stream) {
  if (rows <= 0) return 0;
  if (table_width <= 0 || entries <= 0 || kv_heads <= 0 || q_heads <= 0 || q_heads % kv_heads || page_size <= 0 || num_pages <= 0 ||
      budget <= 0 || static_cast<long long>(budget) * page_size > (1ll << 30) || parts < 1 || parts > 8) return B200_ERR_BAD_SIZE;
  AttendArgs a{q, keys, values, chosen, positions, token_entry, block_table, out, table_width, rows, entries, q_heads, kv_heads,
               page_size, num_pages, budget, parts, scale * 1.44269504088896340736f};
  if (dtype == kF32) return launch_attend(attend_streams_kernel, a, Streams::heads, Streams::threads / 32, stream);
  if (dtype != kBF16) return B200_ERR_BAD_DTYPE;
  if constexpr (kDim <= 128) {
    if (q_heads / kv_heads > 8) return launch_mma<2, 4>(a, stream);
    if (wide) return launch_mma<1, 8>(a, stream);
  }
  return launch_mma<1, 4>(a, stream);
}
