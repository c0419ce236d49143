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
// have: a row always reads its last page, so nobody asks for them.  Each key is read once, 16 bytes a lane: 511 pages of 16 keys,
// 8 heads of 128 in bfloat16, 18.8 MB in 7.7 us (2.4 TB/s; 4.8 us where L2 holds the keys): a launch's ramp and one round of loads.
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
  return min(position / a.page_size, a.table_width - 1) + 1;
}

constexpr int kChooseThreads = 256, kChooseWarps = kChooseThreads / 32;

template <int WARPS> __device__ __forceinline__ void sync_group() {
  if (WARPS == 1) __syncwarp(); else __syncthreads();
}
constexpr int select_words(int warps) { return 256 + 4 * warps + 4; }      // whole 16 bytes

struct Tally {
  uint32_t always, others;      // how many keys are kKeyAlways, how many are candidates
  uint32_t least, most;         // of the candidates
};

// Whether a key is a candidate's.
__device__ __forceinline__ bool is_other(uint32_t key) { return key != kKeyNone && key != kKeyAlways; }

template <int WARPS> __device__ Tally tally_keys(const uint32_t* keys, int count, uint32_t* scratch, int t) {
  uint32_t* per_warp = scratch + 256;
  Tally y{0, 0, 0xffffffffu, 0};
#pragma unroll 4
  for (int i = t; i < count; i += WARPS * 32) {
    const uint32_t key = keys[i];
    y.always += key == kKeyAlways;
    if (is_other(key)) ++y.others, y.least = min(y.least, key), y.most = max(y.most, key);
  }
  y.always = __reduce_add_sync(0xffffffffu, y.always);
  y.others = __reduce_add_sync(0xffffffffu, y.others);
  y.least = __reduce_min_sync(0xffffffffu, y.least);
  y.most = __reduce_max_sync(0xffffffffu, y.most);
  if (WARPS > 1) {
    __syncthreads();
    if ((t & 31) == 0) reinterpret_cast<uint4*>(per_warp)[t >> 5] = make_uint4(y.always, y.others, y.least, y.most);
    __syncthreads();
    y = Tally{0, 0, 0xffffffffu, 0};
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const uint4 v = reinterpret_cast<const uint4*>(per_warp)[w];
      y.always += v.x, y.others += v.y, y.least = min(y.least, v.z), y.most = max(y.most, v.w);
    }
  }
  return y;
}

struct Border {
  uint32_t threshold, wanted;      // take keys above the threshold, and the first `wanted` equal to it
};

// The border of the `wanted` highest candidates (fewer than there are).  It is found digit by digit of eight bits, from the highest bit
// in which the candidates differ at all (scores lie close together: their upper bits say nothing), until the keys of a digit are
// wanted all or none: two rounds as a rule.  WARPS warps take part (t: the thread among them), all of the CTA's or one.
template <int WARPS> __device__ Border find_border(const uint32_t* keys, int count, const Tally& tally, uint32_t wanted, uint32_t* scratch, int t) {
  constexpr int kThreads = WARPS * 32;
  uint32_t* histogram = scratch;
  uint32_t* found = scratch + 256 + 4 * WARPS;      // digit, how many are still wanted among its keys, how many those are
  const int lane = t & 31, warp = t >> 5;
  int high = tally.least == tally.most ? 0 : 32 - __clz(tally.least ^ tally.most);       // bits below this one differ
  uint32_t threshold = wanted == 0 ? kKeyNaN : (high == 32 ? 0u : tally.most >> high << high);
  while (wanted > 0 && high > 0) {
    const int low = max(high - 8, 0);
    const uint32_t digits = (1u << (high - low)) - 1u;
    for (int i = t; i < 256; i += kThreads) histogram[i] = 0;
    sync_group<WARPS>();
#pragma unroll 4
    for (int i = t; i < count; i += kThreads) {
      const uint32_t key = keys[i];
      if (is_other(key) && (high == 32 || key >> high == threshold >> high)) atomicAdd(&histogram[key >> low & digits], 1u);
    }
    sync_group<WARPS>();
    if (warp == 0) {       // lane l holds the digits 255 - 8 l down to 248 - 8 l
      const uint4 upper = reinterpret_cast<const uint4*>(histogram)[63 - 2 * lane], lower = reinterpret_cast<const uint4*>(histogram)[62 - 2 * lane];
      const uint32_t mine[8] = {upper.w, upper.z, upper.y, upper.x, lower.w, lower.z, lower.y, lower.x};
      uint32_t sum = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += mine[i];
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
          if (before < wanted && wanted <= before + mine[i]) found[0] = 255 - 8 * lane - i, found[1] = wanted - before, found[2] = mine[i];
          before += mine[i];
        }
      }
    }
    sync_group<WARPS>();
    threshold |= found[0] << low;
    wanted = found[1];
    high = low;
    if (wanted == found[2]) {                // all keys of this digit: whatever is not below them
      threshold = threshold > 0 ? threshold - 1 : 0;
      wanted = 0;
    }
  }
  return Border{threshold, wanted};
}

// Each warp keeps a run of the indices: what a border may take of the runs before a thread's own.
struct Runs {
  uint32_t more, same;          // above the threshold, and equal to it
};

template <int WARPS> __device__ Runs count_runs(const uint32_t* keys, int count, uint32_t threshold, uint32_t* scratch, int t) {
  constexpr int kThreads = WARPS * 32;
  uint32_t* per_warp = scratch + 256;
  const int lane = t & 31, warp = t >> 5;
  const int run = (count + kThreads - 1) / kThreads * 32;
  const int from = warp * run, to = min(from + run, count);
  Runs y{0, 0};
  if constexpr (WARPS > 1) {     // a single warp has nobody before it
#pragma unroll 4
    for (int i = from + lane; i < to; i += 32) y.more += keys[i] > threshold, y.same += keys[i] == threshold;
    y.more = __reduce_add_sync(0xffffffffu, y.more);
    y.same = __reduce_add_sync(0xffffffffu, y.same);
    __syncthreads();               // what was in per_warp has been read
    if (lane == 0) reinterpret_cast<uint2*>(per_warp)[warp] = make_uint2(y.more, y.same);
    __syncthreads();
    y = Runs{0, 0};
    for (int w = 0; w < warp; ++w) {
      const uint2 v = reinterpret_cast<const uint2*>(per_warp)[w];
      y.more += v.x, y.same += v.y;
    }
  }
  return y;
}

// The indices of the keys that a border takes, `kept` of them, in rising order; -1 behind them up to `budget`.
template <int WARPS> __device__ void write_pages(const uint32_t* keys, int count, const Border& border, Runs runs, int kept, int budget, int* out, int t) {
  constexpr int kThreads = WARPS * 32;
  const int lane = t & 31, warp = t >> 5;
  const int run = (count + kThreads - 1) / kThreads * 32;
  const int from = warp * run, to = min(from + run, count);
  const uint32_t below = (1u << lane) - 1u;
#pragma unroll 4
  for (int i = from; i < to; i += 32) {
    const uint32_t key = i + lane < to ? keys[i + lane] : kKeyNone;
    const bool greater = i + lane < to && key > border.threshold, tie = i + lane < to && key == border.threshold;
    const uint32_t greater_lanes = __ballot_sync(0xffffffffu, greater), tie_lanes = __ballot_sync(0xffffffffu, tie);
    const uint32_t ties_before = runs.same + __popc(tie_lanes & below);
    if (greater || (tie && ties_before < border.wanted)) out[runs.more + __popc(greater_lanes & below) + min(ties_before, border.wanted)] = i + lane;
    runs.more += __popc(greater_lanes);
    runs.same += __popc(tie_lanes);
  }
  for (int i = kept + t; i < budget; i += kThreads) out[i] = -1;
}

// The `budget` highest of keys[0 .. count) that are not kKeyNone, lower indices first among equals.
template <int WARPS> __device__ void select_pages(const uint32_t* keys, int count, int budget, int* out, uint32_t* scratch, int t) {
  const Tally tally = tally_keys<WARPS>(keys, count, scratch, t);
  const int some = tally.always + tally.others;
  Border border{0, 0};
  // the first and the last pages fit into every budget
  if (some > budget) border = find_border<WARPS>(keys, count, tally, budget - tally.always, scratch, t);
  write_pages<WARPS>(keys, count, border, count_runs<WARPS>(keys, count, border.threshold, scratch, t), min(some, budget), budget, out, t);
}

// U and D (see the top of the file).  A NaN gets into the score by way of D.
__device__ __forceinline__ void add_part(float q, double& up, double& down) {
  if (q > 0) up += q; else down += q;
}
template <typename T> __device__ __forceinline__ void parts_of(const T* q, int group, double& up, double& down) {
  up = down = 0;
#pragma unroll 4
  for (int h = 0; h < group; ++h) add_part(to_float<T>(q[h * kDim]), up, down);
}

// Whether a page is held, and whether it is read whatever its score.
__device__ __forceinline__ bool is_held(const ChooseArgs& a, int id) { return id >= 0 && id < a.num_pages; }
__device__ __forceinline__ uint32_t key_of(const ChooseArgs& a, int p, int seen, bool held, double score) {
  return !held ? kKeyNone : (p < a.first || p >= seen - a.last ? kKeyAlways : score_key(score));
}

// How the bounds of a page are spread over lanes that score it: chunk i of lane l is l + i * lanes, of the low and of the high ones.
template <typename T> struct ScoreLanes {
  static constexpr int chunks = kDim * static_cast<int>(sizeof(T)) / 16;
  static constexpr int lanes = chunks % 16 == 0 ? 16 : RowLanes<T>::lanes;
  static constexpr int per_lane = chunks / lanes;
  static constexpr int values = per_lane * Vec<T>::n;
  // pages of a team in flight: a power of two, and no more than its lanes, one of which each page's sum ends in
  static constexpr int wished = per_lane == 1 ? 4 : (per_lane == 2 ? 2 : 1);
  static constexpr int ahead = wished < lanes ? wished : lanes;
  static_assert(lanes % ahead == 0 && lanes * per_lane == chunks);
  static constexpr int at_once = 32 / lanes * ahead;                            // pages of a warp
};

__device__ __forceinline__ void store_in_cluster(uint32_t address, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;\n" ::"r"(address), "r"(v) : "memory");
}

// Single tokens: a cluster per (row, kv head), whose warps share out the pages; a team of lanes holds U and D in registers and reads
// a page's bounds 16 bytes a lane, the next pages' ones before these are summed.  Every score's key goes into the first CTA's shared
// memory, which then chooses.  Scores are summed in 64 bits and rounded once to 32.  The products of bfloat16 numbers are exact there,
// the sums are not once their terms lie further apart than 53 bits: a score next to a midpoint of two 32-bit numbers can come out one
// step apart from the tile kernel's below, which adds in another order.  One request of 2,048 pages 12.5 us (latencies in a row), 32 of
// up to 2,048 pages, 171 MB, 53 us: issue and latency of the 64-bit sums at 14 warps an SM, and rows of unequal length.
template <typename T> __global__ void __launch_bounds__(kChooseThreads, ScoreLanes<T>::values <= 8 ? 2 : 1)
choose_pages_kernel(const __grid_constant__ ChooseArgs a) {
  using L = Vec<T>;
  using R = ScoreLanes<T>;
  constexpr int A = R::ahead;
  extern __shared__ uint32_t keys[];
  __shared__ __align__(16) uint32_t scratch[select_words(kChooseWarps)];
  if (a.cluster > 1) cluster_arrive();
  pdl_trigger();
  pdl_wait();
  const int share = blockIdx.x % a.cluster, unit = blockIdx.x / a.cluster, lane = threadIdx.x & 31;
  const int row = unit / a.kv_heads, head = unit % a.kv_heads;
  const int entry = a.token_entry[row], seen = visible_pages(a, a.positions[row], entry);
  const int from = (share * kChooseWarps + (threadIdx.x >> 5)) * R::at_once, stride = a.cluster * kChooseWarps * R::at_once;
  const int* table = a.block_table + static_cast<size_t>(seen > 0 ? entry : 0) * a.table_width;
  const uint32_t keys_at = a.cluster > 1 ? in_cluster(shared_address(keys), 0) : 0;
  auto put = [&](int p, uint32_t key) {
    if (a.cluster > 1) store_in_cluster(keys_at + p * 4, key); else keys[p] = key;
  };
  if (a.cluster > 1) cluster_wait();          // every CTA of the cluster has started
  if (seen <= a.budget) {                     // nothing to choose from: which pages are held is enough
    for (int p = share * kChooseThreads + threadIdx.x; p < seen; p += a.cluster * kChooseThreads) put(p, is_held(a, table[p]) ? kKeyAlways : kKeyNone);
  } else {
    const int team = lane / R::lanes, part = lane % R::lanes;
    // page j of the team in a round is from + team * A + j; ids are asked for a round before the bounds that they lead to
    int ids[A];
#pragma unroll
    for (int j = 0; j < A; ++j) ids[j] = from + team * A + j < seen ? table[from + team * A + j] : -1;
    typename L::type low[A][R::per_lane], high[A][R::per_lane];
    bool is[A];
    auto fetch = [&]() {
#pragma unroll
      for (int j = 0; j < A; ++j) {
        is[j] = is_held(a, ids[j]);
        const typename L::type* at = reinterpret_cast<const typename L::type*>(
            static_cast<const T*>(a.bounds) + (static_cast<size_t>(is[j] ? ids[j] : 0) * a.kv_heads + head) * 2 * kDim);
#pragma unroll
        for (int i = 0; i < R::per_lane; ++i) low[j][i] = at[part + i * R::lanes], high[j][i] = at[R::chunks + part + i * R::lanes];
      }
    };
    // the row's numbers first: behind the bounds, a full machine's worth of them, they would wait
    const int group = a.q_heads / a.kv_heads;
    const typename L::type* q = reinterpret_cast<const typename L::type*>(static_cast<const T*>(a.q) + (static_cast<size_t>(row) * a.q_heads + head * group) * kDim);
    constexpr int kFirst = 32 / R::per_lane >= 8 ? 4 : 2;      // heads asked for together
    typename L::type first[kFirst][R::per_lane];
#pragma unroll
    for (int h = 0; h < kFirst; ++h) {
#pragma unroll
      for (int i = 0; i < R::per_lane; ++i) first[h][i] = h < group ? q[h * R::chunks + part + i * R::lanes] : typename L::type{};
    }
    fetch();
    double u[R::values], d[R::values];
#pragma unroll
    for (int i = 0; i < R::values; ++i) u[i] = d[i] = 0;
    auto add_head = [&](const typename L::type* row_of_head) {
#pragma unroll
      for (int i = 0; i < R::per_lane; ++i) {
        float v[L::n];
        L::unpack(row_of_head[i], v);
#pragma unroll
        for (int x = 0; x < L::n; ++x) add_part(v[x], u[i * L::n + x], d[i * L::n + x]);
      }
    };
#pragma unroll
    for (int h = 0; h < kFirst; ++h) add_head(first[h]);
    for (int h = kFirst; h < group; ++h) {
      typename L::type more[R::per_lane];
#pragma unroll
      for (int i = 0; i < R::per_lane; ++i) more[i] = q[h * R::chunks + part + i * R::lanes];
      add_head(more);
    }
    // the trip count is the same for all lanes: they exchange sums
    for (int base = from; base < seen; base += stride) {
      double sum[A];
      uint32_t held = 0;
#pragma unroll
      for (int j = 0; j < A; ++j) {
        if (is[j]) held |= 1u << j;
        double other = 0;
        sum[j] = 0;
#pragma unroll
        for (int i = 0; i < R::per_lane; ++i) {
          float lo[L::n], hi[L::n];
          L::unpack(low[j][i], lo);
          L::unpack(high[j][i], hi);
#pragma unroll
          for (int x = 0; x < L::n; ++x) {
            sum[j] = fma(static_cast<double>(hi[x]), u[i * L::n + x], sum[j]);
            other = fma(static_cast<double>(lo[x]), d[i * L::n + x], other);
          }
        }
        sum[j] += other;
      }
      const int next = base + stride + team * A;
#pragma unroll
      for (int j = 0; j < A; ++j) ids[j] = next + j < seen ? table[next + j] : -1;
      // halves of the team add up halves of its pages, until every lane is left with one page (its place among the team's A: `mine`)
      int mine = 0, width = R::lanes / 2;
#pragma unroll
      for (int n = A; n > 1; n /= 2, width /= 2) {
        const bool upper = part & width;
#pragma unroll
        for (int j = 0; j < n / 2; ++j) {
          const double give = upper ? sum[j] : sum[j + n / 2], keep = upper ? sum[j + n / 2] : sum[j];
          sum[j] = keep + __shfl_xor_sync(0xffffffffu, give, width);
        }
        mine += upper ? n / 2 : 0;
      }
#pragma unroll
      for (; width >= 1; width /= 2) sum[0] += __shfl_xor_sync(0xffffffffu, sum[0], width);
      fetch();
      const int p = base + team * A + mine;
      if (part % (R::lanes / A) == 0 && p < seen) put(p, key_of(a, p, seen, held >> mine & 1, sum[0]));
    }
  }
  __syncthreads();
  if (a.cluster > 1) {
    cluster_arrive();
    cluster_wait();
    if (share != 0) return;
  }
  select_pages<kChooseWarps>(keys, seen, a.budget, a.chosen + static_cast<size_t>(unit) * a.budget, scratch, threadIdx.x);
}

// Rows of prompts: a cluster per (eight rows, kv head), the scores as a product [8 rows, 2 d] x [2 d, pages] on the 64-bit tensor
// cores (mma.m8n8k4.f64; d sums and u sums against low and high bounds), so that a bound is read and widened once for eight
// rows.  A lane's four numbers of the sum over channels may be any: it takes the channels of one 16-byte chunk one after the other.
// The CTAs of the cluster share out the pages, then the rows: one warp chooses for a row.  Rows of several entries in one tile are
// scored entry by entry.  874 rows of 640 to 1,024 pages, 8 kv heads of 128: 140 us, the 64-bit tensor pipe 66 % busy (a CTA per row:
// 1,733 us).
constexpr int kTileRows = 8;

__device__ __forceinline__ void mma_f64(double (&c)[2], double a, double b) {
  asm volatile("mma.sync.aligned.m8n8k4.row.col.f64.f64.f64.f64 {%0, %1}, {%2}, {%3}, {%0, %1};\n" : "+d"(c[0]), "+d"(c[1]) : "d"(a), "d"(b));
}

template <typename T> __global__ void __launch_bounds__(kChooseThreads, 2) choose_tile_kernel(const __grid_constant__ ChooseArgs a) {
  using L = Vec<T>;
  constexpr int kChunks = 2 * kDim / L::n, kSteps = kChunks / 4;        // 16-byte chunks of a page's bounds; those of one lane
  extern __shared__ double sums[];                       // [kSteps * L::n][row][lane of four]
  uint32_t* keys = reinterpret_cast<uint32_t*>(sums + 2 * kDim * kTileRows);   // [rows of this CTA][table_width]
  __shared__ __align__(16) uint32_t scratch[kChooseWarps][select_words(1)];
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
    const int steps = most > a.budget ? kSteps : 0;      // no row of these has anything to choose from: which pages are held is enough
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
      for (int step = 0; step < steps; ++step) {
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
            const uint32_t key = key_of(a, p, seen, of >= 0, c[j][x]);
            const uint32_t place = (static_cast<uint32_t>(r % share) * a.table_width + p) * 4;
            if (a.cluster > 1) store_in_cluster(in_cluster(keys_at + place, r / share), key);
            else keys[place / 4] = key;
          }
        }
      }
    }
    r0 = r1;
  }
  __syncthreads();
  if (a.cluster > 1) {
    cluster_arrive();
    cluster_wait();
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

inline bool fits(const ChooseArgs& a) {
  return a.table_width > 0 && a.entries > 0 && a.kv_heads > 0 && a.q_heads > 0 && a.q_heads % a.kv_heads == 0 && a.page_size > 0 &&
         a.num_pages > 0 && a.first >= 0 && a.last >= 1 && a.budget >= a.first + a.last &&
         (a.cluster == 1 || a.cluster == 2 || a.cluster == 4 || a.cluster == 8);
}

// Of this build alone: a static of a template that several loaded libraries share by name would be one for all of them, and the shared
// memory of another head size's kernel would go without its limit being raised.
namespace {

template <typename T> int launch_choose(const ChooseArgs& a, cudaStream_t stream) {
  static DeviceOnce once;
  const long long ctas = static_cast<long long>(a.rows) * a.kv_heads * a.cluster, bytes = static_cast<long long>(a.table_width) * 4;
  if (bytes > kChooseSharedBytes || ctas > 0x7fffffffll) return B200_ERR_TOO_LARGE;
  if (const int status = configure_once(once, choose_pages_kernel<T>, kChooseSharedBytes)) return status;
  launch_clusters(choose_pages_kernel<T>, dim3(static_cast<unsigned>(ctas)), dim3(kChooseThreads), static_cast<size_t>(bytes), a.cluster, stream, a);
  return launch_status();
}

template <typename T> int launch_choose_tiles(const ChooseArgs& a, cudaStream_t stream) {
  static DeviceOnce once;
  const long long ctas = static_cast<long long>((a.rows + kTileRows - 1) / kTileRows) * a.kv_heads * a.cluster;
  const long long bytes = static_cast<long long>(a.table_width) * (kTileRows / a.cluster) * 4 + 2 * kDim * kTileRows * 8;
  if (bytes > kChooseSharedBytes || ctas > 0x7fffffffll) return B200_ERR_TOO_LARGE;
  if (const int status = configure_once(once, choose_tile_kernel<T>, kChooseSharedBytes)) return status;
  launch_clusters(choose_tile_kernel<T>, dim3(static_cast<unsigned>(ctas)), dim3(kChooseThreads), static_cast<size_t>(bytes), a.cluster, stream, a);
  return launch_status();
}

}  // namespace
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

// cluster: CTAs of a cluster that share out a row's pages (1, 2, 4 or 8).
extern "C" int b200_choose_pages(const void* q, const void* bounds, const int* positions, const int* token_entry,
                                 const int* block_table, int table_width, int* chosen, int rows, int entries, int q_heads, int kv_heads,
                                 int page_size, int num_pages, int budget, int first, int last, int cluster, int dtype,
                                 cudaStream_t stream) {
  if (rows <= 0) return 0;
  ChooseArgs a{q, bounds, positions, token_entry, block_table, chosen, table_width, rows, entries, q_heads, kv_heads, page_size,
               num_pages, budget, first, last, cluster};
  if (!fits(a)) return B200_ERR_BAD_SIZE;
  B200_DISPATCH_DTYPE(dtype, T, return launch_choose<T>(a, stream));
  return 0;
}

// The same for rows of prompts, eight to a cluster of `cluster` CTAs (1, 2, 4 or 8).
extern "C" int b200_choose_pages_tiles(const void* q, const void* bounds, const int* positions, const int* token_entry,
                                       const int* block_table, int table_width, int* chosen, int rows, int entries, int q_heads,
                                       int kv_heads, int page_size, int num_pages, int budget, int first, int last, int cluster, int dtype,
                                       cudaStream_t stream) {
  if (rows <= 0) return 0;
  ChooseArgs a{q, bounds, positions, token_entry, block_table, chosen, table_width, rows, entries, q_heads, kv_heads, page_size,
               num_pages, budget, first, last, cluster};
  if (!fits(a)) return B200_ERR_BAD_SIZE;
  B200_DISPATCH_DTYPE(dtype, T, return launch_choose_tiles<T>(a, stream));
  return 0;
}
