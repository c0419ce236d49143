// Which pages of its cache matter to a query: bounds of a page's keys, choice of pages by a cheap score.  One build per head
// size (HEAD_DIM).
//
//   bounds:  low_c(P) = min over the keys k of page P of k_c,   high_c(P) = max
//   score:   s(P) = sum over the heads h of a group and the channels c of max(q_hc low_c, q_hc high_c),
//            an upper bound of sum_h q_h.k for every key k of P.  Since max(q low, q high) is q high for q > 0 and q low for
//            q < 0, the sum over the heads comes first:  s(P) = sum_c high_c U_c + low_c D_c,
//            U = sum_h max(q_h, 0), D = sum_h min(q_h, 0): 2 HEAD_DIM products a page, however many heads the group has.
//   choice:  the first `first` and the last `last` pages that a row sees, of the others those with the highest scores, `budget`
//            in all; of equal scores the lower page.
//   (sparse_attention.cu: softmax(scale q.k) over the keys of the chosen pages at positions up to the row's own.)
//
// Pages are [page][kv head][slot][HEAD_DIM], bounds [page][kv head][low, high][HEAD_DIM], both in the cache's type.
#include "sparse_pages.cuh"

namespace b200 {

template <typename T> __device__ __forceinline__ T min_nan(T a, T b);
template <typename T> __device__ __forceinline__ T max_nan(T a, T b);
template <> __device__ __forceinline__ float min_nan<float>(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
template <> __device__ __forceinline__ float max_nan<float>(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// ----------------------------------------------------------------------------------------------------------- bounds
struct BoundsArgs {
  const void* keys;
  void* bounds;
  const int* block_table;
  const int* q_start;
  const int* kv_len;
  int table_width, entries, kv_heads, page_size, num_pages;
};

// A warp takes (entry, page that this step's tokens fill, kv head) triples.  Pages that are not full keep the bounds they
// have: a row always reads its last page, so nobody asks for them.
template <typename T> __global__ void __launch_bounds__(128) page_bounds_kernel(const __grid_constant__ BoundsArgs a) {
  using L = Vec<T>;
  constexpr int kChunks = RowLanes<T>::chunks;
  constexpr int kCols = kChunks >= 32 ? 32 : (kChunks >= 16 ? 16 : (kChunks >= 8 ? 8 : (kChunks >= 4 ? 4 : 2)));   // lanes across a row
  constexpr int kRows = 32 / kCols;            // rows a warp reads at a time
  pdl_trigger();
  pdl_wait();
  const int r = blockIdx.y, lane = threadIdx.x & 31;
  const int length = a.kv_len[r], count = a.q_start[r + 1] - a.q_start[r];
  if (length <= 0 || count <= 0) return;
  const int from = max(length - count, 0) / a.page_size, to = min(length / a.page_size, a.table_width);
  const int units = (to - from) * a.kv_heads;
  for (int u = blockIdx.x * 4 + (threadIdx.x >> 5); u < units; u += gridDim.x * 4) {
    const int column = from + u / a.kv_heads, head = u % a.kv_heads;
    const int page = a.block_table[static_cast<size_t>(r) * a.table_width + column];
    if (page < 0 || page >= a.num_pages) continue;
    const size_t tile = static_cast<size_t>(page) * a.kv_heads + head;
    const typename L::type* src = reinterpret_cast<const typename L::type*>(static_cast<const T*>(a.keys) + tile * a.page_size * kDim);
    typename L::type* dst = reinterpret_cast<typename L::type*>(static_cast<T*>(a.bounds) + tile * 2 * kDim);
    for (int c0 = 0; c0 < kChunks; c0 += kCols) {
      const int c = c0 + lane % kCols;
      const bool is = kChunks % kCols == 0 || c < kChunks;
      float low[L::n], high[L::n];
#pragma unroll
      for (int i = 0; i < L::n; ++i) low[i] = CUDART_INF_F, high[i] = -CUDART_INF_F;
#pragma unroll 4
      for (int row = is ? lane / kCols : a.page_size; row < a.page_size; row += kRows) {
        float v[L::n];
        L::unpack(src[static_cast<size_t>(row) * kChunks + c], v);
#pragma unroll
        for (int i = 0; i < L::n; ++i) low[i] = min_nan(low[i], v[i]), high[i] = max_nan(high[i], v[i]);
      }
#pragma unroll
      for (int o = kCols; o < 32; o <<= 1) {
#pragma unroll
        for (int i = 0; i < L::n; ++i) {
          low[i] = min_nan(low[i], __shfl_xor_sync(0xffffffffu, low[i], o));
          high[i] = max_nan(high[i], __shfl_xor_sync(0xffffffffu, high[i], o));
        }
      }
      if (is && lane < kCols) dst[c] = L::pack(low), dst[kChunks + c] = L::pack(high);
    }
  }
}

// ----------------------------------------------------------------------------------------------------------- choice
struct ChooseArgs {
  const void* q;
  const void* bounds;
  const int* positions;
  const int* token_entry;
  const int* block_table;
  int* chosen;
  int table_width, rows, entries, q_heads, kv_heads, page_size, num_pages, budget, first, last, cluster;
};

constexpr uint32_t kKeyNone = 0u, kKeyAlways = 0xffffffffu, kKeyNaN = 0xfffffffeu;

// Order-preserving key of a score: larger scores have larger keys, -0 is 0, NaN is above infinity, no score has key 0.
__device__ __forceinline__ uint32_t score_key(double score) {
  const float f = __double2float_rn(score) + 0.f;
  if (f != f) return kKeyNaN;
  const uint32_t u = __float_as_uint(f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Pages that a row sees: 0 for a row that stands nowhere (an entry that is none, a negative position).
__device__ __forceinline__ int visible_pages(const ChooseArgs& a, int position, int entry) {
  if (position < 0 || entry < 0 || entry >= a.entries) return 0;
  return min(position / a.page_size + 1, a.table_width);
}

constexpr int kChooseThreads = 256, kChooseWarps = kChooseThreads / 32;

template <int WARPS> __device__ __forceinline__ void sync_group() {
  if (WARPS == 1) __syncwarp(); else __syncthreads();
}
constexpr int select_words(int warps) { return 256 + 3 * warps + 2; }

// The `budget` highest of keys[0 .. count) that are not kKeyNone, lower indices first among equals, written in rising order
// of their indices; -1 behind them.  WARPS warps take part (t: the thread among them), all of the CTA's or one.
template <int WARPS> __device__ void select_pages(const uint32_t* keys, int count, int budget, int* out, uint32_t* scratch, int t) {
  constexpr int kThreads = WARPS * 32;
  uint32_t* histogram = scratch;
  uint32_t* held = scratch + 256;              // per warp
  uint32_t* above = held + WARPS;
  uint32_t* equal = above + WARPS;
  uint32_t* found = equal + WARPS;             // digit, how many are still wanted among its keys
  const int lane = t & 31, warp = t >> 5;
  uint32_t some = 0;
  for (int i = t; i < count; i += kThreads) some += keys[i] != kKeyNone;
  some = __reduce_add_sync(0xffffffffu, some);
  if (WARPS > 1) {
    if (lane == 0) held[warp] = some;
    __syncthreads();
    some = 0;
    for (int w = 0; w < WARPS; ++w) some += held[w];
  }
  uint32_t threshold = 0, wanted = 0;          // take keys above the threshold, and the first `wanted` equal to it
  if (some > static_cast<uint32_t>(budget)) {
    wanted = budget;
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = t; i < 256; i += kThreads) histogram[i] = 0;
      sync_group<WARPS>();
      for (int i = t; i < count; i += kThreads) {
        const uint32_t key = keys[i];
        if (key != kKeyNone && (shift == 24 || (key >> (shift + 8)) == (threshold >> (shift + 8)))) atomicAdd(&histogram[(key >> shift) & 255u], 1u);
      }
      sync_group<WARPS>();
      if (warp == 0) {       // lane l holds the digits 255 - 8 l down to 248 - 8 l
        uint32_t mine[8], sum = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) mine[i] = histogram[255 - 8 * lane - i], sum += mine[i];
        uint32_t upto = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const uint32_t other = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += other;
        }
        uint32_t before = upto - sum;
        if (before < wanted && wanted <= upto) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if (before < wanted && wanted <= before + mine[i]) found[0] = 255 - 8 * lane - i, found[1] = wanted - before;
            before += mine[i];
          }
        }
      }
      sync_group<WARPS>();
      threshold |= found[0] << shift;
      wanted = found[1];
    }
  }
  // each warp keeps a run of indices: count, then write at the place the warps before it leave
  const int run = (count + kThreads - 1) / kThreads * 32;
  const int from = warp * run, to = min(from + run, count);
  uint32_t more = 0, same = 0;
  if (WARPS > 1) {
    for (int i = from + lane; i < to; i += 32) more += keys[i] > threshold, same += keys[i] == threshold;
    more = __reduce_add_sync(0xffffffffu, more);
    same = __reduce_add_sync(0xffffffffu, same);
    if (lane == 0) above[warp] = more, equal[warp] = same;
    __syncthreads();
    more = same = 0;
    for (int w = 0; w < warp; ++w) more += above[w], same += equal[w];
  }
  const uint32_t below = (1u << lane) - 1u;
  for (int i = from; i < to; i += 32) {
    const uint32_t key = i + lane < to ? keys[i + lane] : kKeyNone;
    const bool greater = i + lane < to && key > threshold, tie = i + lane < to && key == threshold;
    const uint32_t greater_lanes = __ballot_sync(0xffffffffu, greater), tie_lanes = __ballot_sync(0xffffffffu, tie);
    const uint32_t ties_before = same + __popc(tie_lanes & below);
    if (greater || (tie && ties_before < wanted)) out[more + __popc(greater_lanes & below) + min(ties_before, wanted)] = i + lane;
    more += __popc(greater_lanes);
    same += __popc(tie_lanes);
  }
  const int kept = min(some, static_cast<uint32_t>(budget));
  for (int i = kept + t; i < budget; i += kThreads) out[i] = -1;
}

// U and D of one channel (see the top of the file).  A NaN goes into both sums' score by way of D.
template <typename T> __device__ __forceinline__ void parts_of(const T* q, int group, double& up, double& down) {
  up = down = 0;
  for (int h = 0; h < group; ++h) {
    const double v = to_float<T>(q[h * kDim]);
    if (v > 0) up += v; else down += v;
  }
}

__device__ __forceinline__ void store_in_cluster(uint32_t address, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;\n" ::"r"(address), "r"(v) : "memory");
}

// Single tokens: a cluster per (row, kv head).  Its CTAs share out the pages; a few lanes (RowLanes) hold U and D in registers
// and read a page's bounds 16 bytes at a time; every score's key goes into the first CTA's shared memory, which then chooses.
// Scores are summed in 64 bits and rounded once: the products of bfloat16 numbers are exact there, so neither the order of the sum
// nor its spread over lanes moves a page across the border.
template <typename T> __global__ void __launch_bounds__(kChooseThreads, RowLanes<T>::values * sizeof(T) <= 32 ? 2 : 1)
choose_pages_kernel(const __grid_constant__ ChooseArgs a) {
  using L = Vec<T>;
  using R = RowLanes<T>;
  extern __shared__ uint32_t keys[];
  __shared__ double up[kDim], down[kDim];
  __shared__ uint32_t scratch[select_words(kChooseWarps)];
  if (a.cluster > 1) cluster_arrive();
  pdl_trigger();
  pdl_wait();
  const int rank = blockIdx.x % a.cluster, unit = blockIdx.x / a.cluster, t = threadIdx.x;
  const int row = unit / a.kv_heads, head = unit % a.kv_heads;
  const int entry = a.token_entry[row], seen = visible_pages(a, a.positions[row], entry);
  const int group = a.q_heads / a.kv_heads;
  const int* table = a.block_table + static_cast<size_t>(seen > 0 ? entry : 0) * a.table_width;
  for (int c = t; c < kDim; c += kChooseThreads)
    parts_of(static_cast<const T*>(a.q) + (static_cast<size_t>(row) * a.q_heads + head * group) * kDim + c, group, up[c], down[c]);
  __syncthreads();
  constexpr int kTeams = kChooseThreads / R::lanes, kAhead = R::values <= 16 ? 2 : 1;
  const int team = t / R::lanes, part = t % R::lanes, stride = a.cluster * kTeams;
  double u[R::values], d[R::values];
#pragma unroll
  for (int i = 0; i < R::values; ++i) {
    const int c = (part + i / L::n * R::lanes) * L::n + i % L::n;
    u[i] = up[c], d[i] = down[c];
  }
  const uint32_t keys_at = a.cluster > 1 ? in_cluster(shared_address(keys), 0) : 0;
  if (a.cluster > 1) cluster_wait();          // every CTA of the cluster has started
  // the trip count is the same for all threads: the teams of a warp exchange sums
  for (int base = rank * kTeams; base < seen; base += kAhead * stride) {
    typename L::type low[kAhead][R::per_lane], high[kAhead][R::per_lane];
    bool is[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int p = base + j * stride + team, id = p < seen ? table[p] : -1;
      is[j] = id >= 0 && id < a.num_pages;
      const typename L::type* at = reinterpret_cast<const typename L::type*>(
          static_cast<const T*>(a.bounds) + (static_cast<size_t>(is[j] ? id : 0) * a.kv_heads + head) * 2 * kDim);
#pragma unroll
      for (int i = 0; i < R::per_lane; ++i) {
        if (is[j]) low[j][i] = at[part + i * R::lanes], high[j][i] = at[R::chunks + part + i * R::lanes];
        else low[j][i] = high[j][i] = typename L::type{};
      }
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      double sum = 0, other = 0;
#pragma unroll
      for (int i = 0; i < R::per_lane; ++i) {
        float lo[L::n], hi[L::n];
        L::unpack(low[j][i], lo);
        L::unpack(high[j][i], hi);
#pragma unroll
        for (int x = 0; x < L::n; ++x) {
          sum = fma(static_cast<double>(hi[x]), u[i * L::n + x], sum);
          other = fma(static_cast<double>(lo[x]), d[i * L::n + x], other);
        }
      }
      sum += other;
#pragma unroll
      for (int o = 1; o < R::lanes; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      const int p = base + j * stride + team;
      if (part == 0 && p < seen) {
        const uint32_t key = !is[j] ? kKeyNone : (p < a.first || p >= seen - a.last ? kKeyAlways : score_key(sum));
        if (a.cluster > 1) store_in_cluster(keys_at + p * 4, key); else keys[p] = key;
      }
    }
  }
  if (a.cluster > 1) {
    cluster_arrive();
    if (rank != 0) {        // the first CTA is still there: it leaves after this barrier only
      cluster_wait();
      return;
    }
    cluster_wait();
  } else {
    __syncthreads();
  }
  select_pages<kChooseWarps>(keys, seen, a.budget, a.chosen + static_cast<size_t>(unit) * a.budget, scratch, t);
}

// Rows of prompts: a cluster per (eight rows, kv head), the scores as a product [8 rows, 2 d] x [2 d, pages] on the 64-bit tensor
// cores (mma.m8n8k4.f64; d sums and u sums against low and high bounds), so that a bound is read and widened once for eight
// rows.  A lane's four numbers of the sum over channels may be any: it takes the channels of one 16-byte chunk one after the other.
// The CTAs of the cluster share out the pages, then the rows: one warp chooses for a row.  Rows of several entries in one tile are
// scored entry by entry.
constexpr int kTileRows = 8;

__device__ __forceinline__ void mma_f64(double (&c)[2], double a, double b) {
  asm volatile("mma.sync.aligned.m8n8k4.row.col.f64.f64.f64.f64 {%0, %1}, {%2}, {%3}, {%0, %1};\n" : "+d"(c[0]), "+d"(c[1]) : "d"(a), "d"(b));
}

template <typename T> __global__ void __launch_bounds__(kChooseThreads, 2) choose_tile_kernel(const __grid_constant__ ChooseArgs a) {
  using L = Vec<T>;
  constexpr int kChunks = 2 * kDim / L::n, kSteps = kChunks / 4;        // 16-byte chunks of a page's bounds; those of one lane
  extern __shared__ double sums[];                       // [kSteps * L::n][row][lane of four]
  uint32_t* keys = reinterpret_cast<uint32_t*>(sums + 2 * kDim * kTileRows);   // [rows of this CTA][table_width]
  __shared__ uint32_t scratch[kChooseWarps][select_words(1)];
  __shared__ int entries[kTileRows], seens[kTileRows];
  if (a.cluster > 1) cluster_arrive();
  pdl_trigger();
  pdl_wait();
  const int rank = blockIdx.x % a.cluster, unit = blockIdx.x / a.cluster, t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const int head = unit % a.kv_heads, row0 = unit / a.kv_heads * kTileRows, here = min(kTileRows, a.rows - row0);
  const int group = a.q_heads / a.kv_heads, share = kTileRows / a.cluster;
  if (t < kTileRows) {
    const int entry = t < here ? a.token_entry[row0 + t] : -1;
    entries[t] = entry;
    seens[t] = t < here ? visible_pages(a, a.positions[row0 + t], entry) : 0;
  }
  for (int i = t; i < kTileRows * kDim; i += kChooseThreads) {
    const int r = i / kDim, c = i % kDim;
    double up = 0, down = 0;
    if (r < here) parts_of(static_cast<const T*>(a.q) + (static_cast<size_t>(row0 + r) * a.q_heads + head * group) * kDim + c, group, up, down);
    // channel c lies in chunk c / n of the low bounds and as far behind those in the high ones
    const int low = c / L::n, high = low + kChunks / 2;
    sums[((low / 4 * L::n + c % L::n) * kTileRows + r) * 4 + low % 4] = down;
    sums[((high / 4 * L::n + c % L::n) * kTileRows + r) * 4 + high % 4] = up;
  }
  __syncthreads();
  if (a.cluster > 1) cluster_wait();          // every CTA of the cluster has started
  const uint32_t keys_at = shared_address(keys);
  for (int r0 = 0; r0 < here;) {
    const int entry = entries[r0];
    int r1 = r0, most = 0;
    while (r1 < here && entries[r1] == entry) most = max(most, seens[r1++]);
    const int* table = a.block_table + static_cast<size_t>(most > 0 ? entry : 0) * a.table_width;
    for (int p0 = (rank * kChooseWarps + warp) * 16; p0 < most; p0 += a.cluster * kChooseWarps * 16) {
      int id[2];
      const typename L::type* at[2];
      double c[2][2] = {};
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int p = p0 + 8 * j + (lane >> 2);
        id[j] = p < most ? table[p] : -1;
        if (id[j] >= a.num_pages) id[j] = -1;
        at[j] = reinterpret_cast<const typename L::type*>(static_cast<const T*>(a.bounds) + (static_cast<size_t>(max(id[j], 0)) * a.kv_heads + head) * 2 * kDim) + (lane & 3);
      }
#pragma unroll 4
      for (int step = 0; step < kSteps; ++step) {
        float b[2][L::n];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          typename L::type v{};
          if (id[j] >= 0) v = at[j][4 * step];
          L::unpack(v, b[j]);
        }
#pragma unroll
        for (int x = 0; x < L::n; ++x) {
          const double s = sums[(step * L::n + x) * 32 + lane];
#pragma unroll
          for (int j = 0; j < 2; ++j) mma_f64(c[j], s, static_cast<double>(b[j][x]));
        }
      }
      const int r = lane >> 2, seen = seens[r];       // the row that this lane has scores of; pages 2 (lane % 4) and the next
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int of = __shfl_sync(0xffffffffu, id[j], (2 * (lane & 3) + x) * 4), p = p0 + 8 * j + 2 * (lane & 3) + x;
          if (r >= r0 && r < r1 && p < seen) {
            const uint32_t key = of < 0 ? kKeyNone : (p < a.first || p >= seen - a.last ? kKeyAlways : score_key(c[j][x]));
            const uint32_t place = (static_cast<uint32_t>(r % share) * a.table_width + p) * 4;
            if (a.cluster > 1) store_in_cluster(in_cluster(keys_at + place, r / share), key);
            else keys[place / 4] = key;
          }
        }
      }
    }
    r0 = r1;
  }
  if (a.cluster > 1) {
    cluster_arrive();
    cluster_wait();
  } else {
    __syncthreads();
  }
  const int r = rank * share + warp;
  if (warp < share && r < here)
    select_pages<1>(keys + static_cast<size_t>(warp) * a.table_width, seens[r], a.budget,
                    a.chosen + (static_cast<size_t>(row0 + r) * a.kv_heads + head) * a.budget, scratch[warp], lane);
}

template <typename T> int launch_bounds_kernel(const BoundsArgs& a, int max_full, cudaStream_t stream) {
  const int blocks = (max_full * a.kv_heads + 3) / 4;
  launch(page_bounds_kernel<T>, dim3(blocks, a.entries), dim3(128), 0, stream, a);
  return launch_status();
}

constexpr int kChooseSharedBytes = 200 * 1024;

// tile: eight rows to a cluster
template <typename T> int launch_choose(const ChooseArgs& a, int tile, cudaStream_t stream) {
  static DeviceOnce once, once_tile;
  const long long units = static_cast<long long>(tile ? (a.rows + kTileRows - 1) / kTileRows : a.rows) * a.kv_heads;
  const long long words = static_cast<long long>(a.table_width) * (tile ? kTileRows / a.cluster : 1);
  const long long bytes = words * 4 + (tile ? 2 * kDim * kTileRows * 8 : 0);
  if (bytes > kChooseSharedBytes || units * a.cluster > 0x7fffffffll) return B200_ERR_TOO_LARGE;
  const auto kernel = tile ? choose_tile_kernel<T> : choose_pages_kernel<T>;
  if (const int status = configure_once(tile ? once_tile : once, kernel, kChooseSharedBytes)) return status;
  launch_clusters(kernel, dim3(static_cast<unsigned>(units * a.cluster)), dim3(kChooseThreads), static_cast<size_t>(bytes), a.cluster, stream, a);
  return launch_status();
}

}  // namespace b200

using namespace b200;

extern "C" int b200_sparse_pages_head_dim() { return kDim; }

extern "C" int b200_page_bounds(const void* keys, void* bounds, const int* block_table, int table_width, const int* q_start,
                                const int* kv_len, int entries, int max_full, int kv_heads, int page_size, int num_pages, int dtype,
                                cudaStream_t stream) {
  if (entries <= 0 || max_full <= 0) return 0;
  if (table_width <= 0 || kv_heads <= 0 || page_size <= 0 || num_pages <= 0 || entries > 65535) return B200_ERR_BAD_SIZE;
  BoundsArgs a{keys, bounds, block_table, q_start, kv_len, table_width, entries, kv_heads, page_size, num_pages};
  B200_DISPATCH_DTYPE(dtype, T, return launch_bounds_kernel<T>(a, max_full, stream));
  return 0;
}

extern "C" int b200_choose_pages(const void* q, const void* bounds, const int* positions, const int* token_entry,
                                 const int* block_table, int table_width, int* chosen, int rows, int entries, int q_heads, int kv_heads,
                                 int page_size, int num_pages, int budget, int first, int last, int tile, int cluster, int dtype, cudaStream_t stream) {
  if (rows <= 0) return 0;
  if (table_width <= 0 || entries <= 0 || kv_heads <= 0 || q_heads <= 0 || q_heads % kv_heads || page_size <= 0 || num_pages <= 0 ||
      first < 0 || last < 1 || budget < first + last || (cluster != 1 && cluster != 2 && cluster != 4 && cluster != 8)) return B200_ERR_BAD_SIZE;
  ChooseArgs a{q, bounds, positions, token_entry, block_table, chosen, table_width, rows, entries, q_heads, kv_heads, page_size,
               num_pages, budget, first, last, cluster};
  B200_DISPATCH_DTYPE(dtype, T, return launch_choose<T>(a, tile, stream));
  return 0;
}
