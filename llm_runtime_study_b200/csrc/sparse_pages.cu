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
  int table_width, rows, entries, q_heads, kv_heads, page_size, num_pages, budget, first, last;
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

constexpr int kChooseThreads = 256;

// The `budget` highest of keys[0 .. count) that are not kKeyNone, lower indices first among equals, written in rising order
// of their indices; -1 behind them.  All threads of the CTA; scratch: 256 + 3 * warps + 4 words.
__device__ void select_pages(const uint32_t* keys, int count, int budget, int* out, uint32_t* scratch) {
  constexpr int kWarps = kChooseThreads / 32;
  uint32_t* histogram = scratch;
  uint32_t* held = scratch + 256;              // per warp
  uint32_t* above = held + kWarps;
  uint32_t* equal = above + kWarps;
  uint32_t* found = equal + kWarps;            // digit, how many are still wanted among its keys
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  uint32_t some = 0;
  for (int i = t; i < count; i += kChooseThreads) some += keys[i] != kKeyNone;
  some = __reduce_add_sync(0xffffffffu, some);
  if (lane == 0) held[warp] = some;
  __syncthreads();
  some = 0;
  for (int w = 0; w < kWarps; ++w) some += held[w];
  uint32_t threshold = 0, wanted = 0;          // take keys above the threshold, and the first `wanted` equal to it
  if (some > static_cast<uint32_t>(budget)) {
    wanted = budget;
    for (int shift = 24; shift >= 0; shift -= 8) {
      histogram[t] = 0;
      __syncthreads();
      for (int i = t; i < count; i += kChooseThreads) {
        const uint32_t key = keys[i];
        if (key != kKeyNone && (shift == 24 || (key >> (shift + 8)) == (threshold >> (shift + 8)))) atomicAdd(&histogram[(key >> shift) & 255u], 1u);
      }
      __syncthreads();
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
      __syncthreads();
      threshold |= found[0] << shift;
      wanted = found[1];
    }
  }
  // each warp keeps a run of indices: count, then write at the place the warps before it leave
  const int run = (count + kWarps * 32 - 1) / (kWarps * 32) * 32;
  const int from = warp * run, to = min(from + run, count);
  uint32_t more = 0, same = 0;
  for (int i = from + lane; i < to; i += 32) more += keys[i] > threshold, same += keys[i] == threshold;
  more = __reduce_add_sync(0xffffffffu, more);
  same = __reduce_add_sync(0xffffffffu, same);
  if (lane == 0) above[warp] = more, equal[warp] = same;
  __syncthreads();
  more = same = 0;
  for (int w = 0; w < warp; ++w) more += above[w], same += equal[w];
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
  for (int i = kept + t; i < budget; i += kChooseThreads) out[i] = -1;
}

// One CTA per (row, kv head): the scores of all its pages into shared memory, then the choice.  Scores are summed in 64 bits
// and rounded once: the products of bfloat16 numbers are exact there, so neither the order of the sum nor the spread over
// lanes moves a page across the border.
template <typename T> __global__ void __launch_bounds__(kChooseThreads) choose_pages_kernel(const __grid_constant__ ChooseArgs a) {
  using L = Vec<T>;
  using R = RowLanes<T>;
  extern __shared__ uint32_t keys[];
  __shared__ double up[kDim], down[kDim];
  __shared__ uint32_t scratch[256 + 3 * (kChooseThreads / 32) + 4];
  pdl_trigger();
  pdl_wait();
  const int row = blockIdx.x / a.kv_heads, head = blockIdx.x % a.kv_heads, t = threadIdx.x;
  const int entry = a.token_entry[row], seen = visible_pages(a, a.positions[row], entry);
  const int group = a.q_heads / a.kv_heads;
  const int* table = a.block_table + static_cast<size_t>(seen > 0 ? entry : 0) * a.table_width;
  for (int c = t; c < kDim; c += kChooseThreads) {
    const T* q = static_cast<const T*>(a.q) + (static_cast<size_t>(row) * a.q_heads + head * group) * kDim + c;
    double u = 0, d = 0;
    for (int h = 0; h < group; ++h) {
      const double v = to_float<T>(q[h * kDim]);
      if (v > 0) u += v; else d += v;        // a NaN goes into both sums by way of this one and the score
    }
    up[c] = u, down[c] = d;
  }
  __syncthreads();
  constexpr int kTeams = kChooseThreads / R::lanes;
  const int team = t / R::lanes, part = t % R::lanes;
  for (int p = team; p < (seen + kTeams - 1) / kTeams * kTeams; p += kTeams) {
    const int id = p < seen ? table[p] : -1;
    const bool is = id >= 0 && id < a.num_pages;
    double sum = 0;
    if (is) {
      const typename L::type* low = reinterpret_cast<const typename L::type*>(
          static_cast<const T*>(a.bounds) + (static_cast<size_t>(id) * a.kv_heads + head) * 2 * kDim);
#pragma unroll
      for (int i = 0; i < R::per_lane; ++i) {
        const int chunk = part + i * R::lanes;
        float lo[L::n], hi[L::n];
        L::unpack(low[chunk], lo);
        L::unpack(low[R::chunks + chunk], hi);
#pragma unroll
        for (int j = 0; j < L::n; ++j) {
          sum = fma(static_cast<double>(hi[j]), up[chunk * L::n + j], sum);
          sum = fma(static_cast<double>(lo[j]), down[chunk * L::n + j], sum);
        }
      }
    }
#pragma unroll
    for (int o = 1; o < R::lanes; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (part == 0 && p < seen) keys[p] = !is ? kKeyNone : (p < a.first || p >= seen - a.last ? kKeyAlways : score_key(sum));
  }
  __syncthreads();
  select_pages(keys, seen, a.budget, a.chosen + static_cast<size_t>(blockIdx.x) * a.budget, scratch);
}

template <typename T> int launch_bounds_kernel(const BoundsArgs& a, int max_full, cudaStream_t stream) {
  const int blocks = (max_full * a.kv_heads + 3) / 4;
  launch(page_bounds_kernel<T>, dim3(blocks, a.entries), dim3(128), 0, stream, a);
  return launch_status();
}

template <typename T> int launch_choose(const ChooseArgs& a, cudaStream_t stream) {
  static DeviceOnce once;
  const int bytes = a.table_width * 4;
  if (bytes > 200 * 1024) return B200_ERR_TOO_LARGE;
  if (const int status = configure_once(once, choose_pages_kernel<T>, 200 * 1024)) return status;
  launch(choose_pages_kernel<T>, dim3(a.rows * a.kv_heads), dim3(kChooseThreads), bytes, stream, a);
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
                                 int page_size, int num_pages, int budget, int first, int last, int dtype, cudaStream_t stream) {
  if (rows <= 0) return 0;
  if (table_width <= 0 || entries <= 0 || kv_heads <= 0 || q_heads <= 0 || q_heads % kv_heads || page_size <= 0 || num_pages <= 0 ||
      first < 0 || last < 1 || budget < first + last) return B200_ERR_BAD_SIZE;
  ChooseArgs a{q, bounds, positions, token_entry, block_table, chosen, table_width, rows, entries, q_heads, kv_heads, page_size,
               num_pages, budget, first, last};
  B200_DISPATCH_DTYPE(dtype, T, return launch_choose<T>(a, stream));
  return 0;
}
