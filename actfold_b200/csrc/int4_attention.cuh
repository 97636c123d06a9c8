// What the attention kernels over the 4-bit cache share: which keys the rows of
// a request can see, the list of work and its split over the CTAs, the joins
// of rows that several CTAs worked on.
#pragma once

#include <atomic>
#include <string>

#include "int4_cache.cuh"
#include "tree.cuh"

namespace af {

int attention_patience();  // tree_attention.cu: af_tree_attention_wait_limit sets it for all tree attention, and for the attention weights

namespace kv4 {

constexpr int kPlans = 4;           // segments planned ahead in shared memory
constexpr float kUnset = -3.0e38f;  // reference maximum of a row that has seen no key
constexpr float kRaise = 8.f;       // log2 headroom before a reference maximum is raised
// A reference maximum is set this far (log2) below the score that it is taken from: fp16 probabilities then reach down to
// 2^-31 of the largest one (see tree_attention.cuh). bf16 has fp32's range.
template <int DT>
constexpr float kLead = DT == AF_DTYPE_F16 ? 7.f : 0.f;

struct Params {
  const char *q, *k, *v;                        // 16-bit rows of the step's nodes
  int64_t q_n, q_h, k_n, k_h, v_n, v_h;         // byte strides: node, head
  const char* data;                             // the 4-bit cache
  int64_t d_page, d_head;
  const int *tables, *lengths, *starts;
  const uint32_t* mask;
  int64_t tables_ld, mask_ld;
  int words, batch, total, heads, kv_heads, group, pages, page;
  uint32_t page_mul;                            // see entry_of
  int page_shift;
  int64_t capacity;                             // tokens that a table row can hold
  int window, sinks;                            // window 0: all of the prefix is visible
  int reach;                                    // tokens of the prefix that a window can hold: all, of a chain, whose nodes see themselves, one less
  float scale;                                  // times log2(e); of the attention kernels positive: q is flipped, or made 0, instead
  uint32_t q_flip, q_keep;                      // q = (q ^ flip) & keep, in pairs
  char* out;
  int64_t out_n, out_h;
  float* lse;
  int rows;                                     // of a row tile: consecutive (node, head of the group) pairs of a request
  int row_cost;                                 // of a row tile besides its units
  int whole, whole_long;                        // a row tile of at most this many units is not shared by CTAs; where shares are long
  int least;                                    // units of a share
  int joins;                                    // may a row tile be shared?
  char* ws;
  unsigned* status;
  int patience;                                 // attempts of a wait before it gives up
};

// place / p.page, for places up to 2^30 and pages of 8 d tokens: with s = ceil(log2 d) and m = ceil(2^(31 + s) / d) < 2^32 it is
// (2 (place / 8) m) >> (32 + s), since m is too large by less than d / 2^(31 + s) and place / 8 < 2^27.
__device__ __forceinline__ int entry_of(const Params& p, int place) {
  return (int)(__umulhi((uint32_t)(place >> 3) << 1, p.page_mul) >> p.page_shift);
}
inline void set_page(Params& p, int64_t page) {
  const uint64_t d = (uint64_t)page / kBlockTokens;
  p.page = (int)page;
  p.page_shift = 0;
  while ((1ull << p.page_shift) < d) ++p.page_shift;
  p.page_mul = (uint32_t)(((1ull << (31 + p.page_shift)) + d - 1) / d);
}

// A request's nodes and the units of UNIT keys that any of its rows can see: those of the first tokens, those of the
// window, then those of its own tree.
template <int UNIT>
struct Request {
  int s0, n, len;
  int sink_units, from, cached, units;  // unit x < sink_units lies at place UNIT x, x < cached at UNIT (x - sink_units + from), others are nodes
  int tiles, cost;                      // row tiles, and the cost of one; no cost where there is nothing to do or the values are bad
  bool bad;
};

template <int UNIT>
__device__ __forceinline__ Request<UNIT> request(const Params& p, int b) {
  Request<UNIT> r;
  const int s0 = p.starts[b], s1 = p.starts[b + 1];
  r.len = p.lengths[b];
  r.bad = s0 < 0 || s1 < s0 || s1 > p.total || r.len < 0 || r.len > p.capacity || (p.mask && s1 - s0 > 32 * (int64_t)p.words);
  r.s0 = s0;
  r.n = r.bad ? 0 : s1 - s0;
  const int all = (r.len + UNIT - 1) / UNIT;
  r.sink_units = r.from = 0;
  if (p.window) {
    r.sink_units = (min(p.sinks, r.len) + UNIT - 1) / UNIT;
    r.from = max(r.sink_units, max(0, r.len - p.reach) / UNIT);
  }
  r.cached = r.sink_units + max(0, all - r.from);
  r.units = r.cached + (r.n + UNIT - 1) / UNIT;
  r.tiles = (int)(((int64_t)r.n * p.group + p.rows - 1) / p.rows);
  r.cost = r.n ? r.units + p.row_cost : 0;
  return r;
}

// The list of row tiles, cut into one share per CTA: the first `more` shares have each + 1 units. Short lists are cut into
// shares of p.least units, for as many CTAs as that takes: a part of a row costs its CTA and the join more than a few units do.
struct Shares {
  int each, more, all;
  __device__ __forceinline__ int begin(int i) const { return (int)min((int64_t)all, (int64_t)each * i + min(i, more)); }
  __device__ __forceinline__ int owner(int t) const {
    const int big = more * (each + 1);
    return t < big ? t / (each + 1) : more + (t - big) / each;
  }
};

// The units [x0, x1) of one row tile that a CTA works on (x1 = 0: the share is done).
struct __align__(16) Segment {
  int s0, n, len, b;
  int kvh, row0, x0, x1;               // row0: the tile's first row, counted from the request's first
  int sink_units, from, cached, j0;    // j0: units of the CTA before this segment
  int whole, last;                     // all units of the row?; the CTA with the row's last unit, where this one begins a row that others go on with
  int pad[2];
};

// What CTA c left for the join: it began a row tile that CTAs c + 1 .. last went on with (last = 0: it did not).
struct Started {
  int last, s0, row0, rows, kvh;
};

// One warp plans: its CTA's share [t, end) of the list, cut into segments.
template <int UNIT>
struct Planner {
  Shares shares;
  int t, end, before, b, j;  // units of the requests before b; of the CTA so far
  int whole;                 // a row tile of at most this many units is not shared: fewer where shares are long, which it would make uneven
  Request<UNIT> r;

  __device__ __forceinline__ static int cost_of(const Params& p, int b, bool& disorder) {
    if (b >= p.batch) return 0;
    const Request<UNIT> r = request<UNIT>(p, b);
    disorder |= p.starts[b + 1] < p.starts[b];
    if (r.bad && blockIdx.x == 0 && p.status) atomicOr(p.status, AF_STATUS_BOUNDS);
    return r.cost * r.tiles * p.kv_heads;
  }

  // Two passes over the requests, 32 at a time: the list's length, and the request that the share begins with. Starts out
  // of order anywhere are trees that overlap, whose units nothing bounds: then there is no list.
  __device__ __forceinline__ void begin(const Params& p, int lane) {
    bool disorder = false;
    const int first_cost = cost_of(p, lane, disorder);
    int all = first_cost;
#pragma unroll 4
    for (int x = lane + 32; x < p.batch; x += 32) all += cost_of(p, x, disorder);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
    if (__any_sync(0xffffffffu, disorder)) all = 0;
    shares.all = all;
    shares.each = all / (int)gridDim.x;
    shares.more = all - shares.each * (int)gridDim.x;
    whole = shares.each >= 2 * p.whole ? p.whole_long : p.whole;
    if (shares.each < p.least) shares.each = p.least, shares.more = 0;
    t = shares.begin(blockIdx.x);
    end = shares.begin(blockIdx.x + 1);
    b = before = j = 0;
    if (t >= end) return;
#pragma unroll 1
    for (int b0 = 0; b0 < p.batch; b0 += 32) {
      int upto = b0 ? cost_of(p, b0 + lane, disorder) : first_cost;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
      }
      const uint32_t behind = __ballot_sync(0xffffffffu, t < before + upto);  // lanes whose request ends behind t
      if (behind) {
        const int x = __ffs(behind) - 1;
        b = b0 + x;
        before += x ? __shfl_sync(0xffffffffu, upto, x - 1) : 0;
        break;
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
    r = request<UNIT>(p, b);
  }

  // The share's next segment. A row of up to p.whole units belongs to the CTA whose share it begins in.
  __device__ __forceinline__ bool next(const Params& p, Segment& s) {
#pragma unroll 1
    while (t < end) {
#pragma unroll 1
      while (t >= before + r.cost * r.tiles * p.kv_heads) {
        before += r.cost * r.tiles * p.kv_heads;
        r = request<UNIT>(p, ++b);
      }
      const int row = (t - before) / r.cost, u = (t - before) - row * r.cost;  // (head, row tile), and the place in it
      s.kvh = row / r.tiles;
      s.row0 = (row - s.kvh * r.tiles) * p.rows;
      s.s0 = r.s0, s.n = r.n, s.len = r.len, s.b = b;
      s.sink_units = r.sink_units, s.from = r.from, s.cached = r.cached;
      const bool alone = r.units <= whole;
      const int row_end = t - u + r.cost, upto = alone ? r.cost : min(r.cost, u + (end - t));
      t += upto - u;
      s.x0 = max(0, u - p.row_cost);
      s.x1 = upto - p.row_cost;
      if (alone ? u > 0 : s.x1 <= s.x0) continue;  // begun by another CTA; no unit in this share
      s.whole = s.x0 == 0 && s.x1 == r.units;
      s.last = !s.whole && s.x0 == 0 ? shares.owner(row_end - 1) : 0;
      s.j0 = j;
      j += s.x1 - s.x0;
      return true;
    }
    s.x1 = 0;
    return false;
  }
};

// Bounded wait for a phase: failed[0] says that a wait has run out somewhere, failed[1] how many attempts a wait makes
// (each sleeps a few microseconds; kPatience of them take about a second).
constexpr int kPatience = 1 << 18;
__device__ __forceinline__ bool wait_for(uint32_t bar, uint32_t parity, volatile int* failed) {
#pragma unroll 1
  for (int n = 0; !mbar_try_wait(bar, parity); ++n)
    if (n >= failed[1] || *failed) return false;
  return true;
}

template <int THREADS>
__device__ __forceinline__ bool vote_any(int bar, bool mine) {
  int r;
  asm volatile(
      "{\n\t.reg .pred a, b;\n\t"
      "setp.ne.s32 a, %1, 0;\n\t"
      "barrier.cta.red.or.pred b, %2, %3, a;\n\t"
      "selp.s32 %0, 1, 0, b;\n\t}"
      : "=r"(r)
      : "r"((int)mine), "r"(bar), "n"(THREADS)
      : "memory");
  return r != 0;
}

__device__ __forceinline__ float ex2(float x) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x));
  return e;
}

template <int DT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (DT == AF_DTYPE_BF16) {
    return bits_of(__floats2bfloat162_rn(lo, hi));
  } else {
    return bits_of(__floats2half2_rn(lo, hi));
  }
}

template <int DT>
__device__ __forceinline__ bool not_finite(uint32_t bits) {
  constexpr uint32_t e = DT == AF_DTYPE_BF16 ? 0x7f80u : 0x7c00u;
  return (bits & e) == e;
}
template <int DT>
__device__ __forceinline__ float from_bits(uint32_t bits) {
  const uint16_t b = (uint16_t)bits;
  return load_scalar<DT>(reinterpret_cast<const char*>(&b), 0);
}

// Nodes j0 .. j0 + 31 of the tree (n nodes from s0 on, behind len cached tokens) that node i sees, as bits. j0 is a multiple of 32.
// A chain goes on where the cache ends: the first `sinks` tokens stay visible wherever they lie.
__device__ __forceinline__ uint32_t seen_nodes(const Params& p, int s0, int n, int len, int i, int j0) {
  auto below = [](int x) { return x <= 0 ? 0u : x >= 32 ? 0xffffffffu : (1u << x) - 1u; };
  if (p.mask) return p.mask[(int64_t)(s0 + i) * p.mask_ld + (j0 >> 5)] & below(n - j0);
  return below(i + 1 - j0) & (p.window ? ~below(i + 1 - p.window - j0) | below(p.sinks - len - j0) : 0xffffffffu);
}

// The first place behind the sinks that node i sees: its window holds the nodes that it sees, and then the last tokens of the prefix.
__device__ __forceinline__ int first_place(const Params& p, int s0, int n, int len, int i) {
  if (!p.window) return 0;
  int count = min(i + 1, p.window);
  if (p.mask) {
    count = 0;
#pragma unroll 1
    for (int j = 0; j < n && count < p.window; j += 32) count += __popc(seen_nodes(p, s0, n, len, i, j));
  }
  return max(0, len - max(0, p.window - count));
}

// Workspace: Started[ctas], then per CTA two partial row tiles (0: begun by an earlier CTA, 1: begun here) of [N][HD] fp32 sums
// and [N] (maximum, sum) pairs.
template <int N, int HD>
struct Scratch {
  char* base;
  int ctas;
  static constexpr int64_t kHead = 32;
  static_assert(sizeof(Started) <= kHead, "one Started per CTA");
  __host__ __device__ static int64_t bytes(int ctas) { return ctas * (kHead + (int64_t)2 * N * (HD + 2) * 4); }
  __device__ Started* started(int c) const { return reinterpret_cast<Started*>(base + c * kHead); }
  __device__ float* sums(int c, int which) const { return reinterpret_cast<float*>(base + ctas * kHead) + ((int64_t)c * 2 + which) * N * HD; }
  __device__ float2* stats(int c, int which) const {
    return reinterpret_cast<float2*>(base + ctas * (kHead + (int64_t)2 * N * HD * 4)) + ((int64_t)c * 2 + which) * N;
  }
};

constexpr int kWideUnit = 128;
// The kernel for many rows (int4_attention_wide.cu).
int wide_launch(const Params& p, bool bf16, int head_dim, cudaStream_t s);

template <auto Kernel>
int allow_smem(int bytes, const char* what) {
  static std::atomic<uint64_t> allowed{0};  // a bit per device
  int device = 0;
  cudaGetDevice(&device);
  const uint64_t bit = 1ull << (device & 63);
  if (allowed.load(std::memory_order_relaxed) & bit) return AF_OK;
  const cudaError_t e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return fail(AF_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
  allowed.fetch_or(bit, std::memory_order_relaxed);
  return AF_OK;
}

constexpr int kJoinThreads = 256;

// Rows that several CTAs worked on: out = sum_c w_c O_c / sum_c w_c l_c with w_c = 2^(m_c - max m), in the CTAs' order. The
// block's 8 warps share a row's parts where there are many, and take a row each where there are few.
template <int DT, int N, int HD>
__global__ void __launch_bounds__(kJoinThreads) k_join(const __grid_constant__ Params p, int ctas) {
  constexpr int V = HD / 32, W = kJoinThreads / 32;
  __shared__ float acc[W][HD + 1];
  pdl_wait();
  const Scratch<N, HD> scratch{p.ws, ctas};
  const int c = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Started st = *scratch.started(c);
  if (st.last <= c) return;
  const int parts = st.last - c + 1;
  const bool share = parts > 8;
  for (int row = share ? blockIdx.y : blockIdx.y * W + warp; row < st.rows; row += share ? gridDim.y : gridDim.y * W) {
    float m = kUnset;
    for (int i = lane; i < parts; i += 32) m = fmaxf(m, scratch.stats(c + i, i == 0)[row].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    float sum = 0.f, y[V];
#pragma unroll
    for (int v = 0; v < V; ++v) y[v] = 0.f;
#pragma unroll 4
    for (int i = share ? warp : 0; i < parts; i += share ? W : 1) {
      const float2 ml = scratch.stats(c + i, i == 0)[row];
      const float w = ml.x == m ? 1.f : exp2f(ml.x - m);
      const float* o = scratch.sums(c + i, i == 0) + (int64_t)row * HD + lane * V;
      sum += w * ml.y;
#pragma unroll
      for (int v = 0; v < V; ++v) y[v] += w * o[v];  // (a part without a key has weight 0 and sums of 0)
    }
    if (share) {
      __syncthreads();
#pragma unroll
      for (int v = 0; v < V; ++v) acc[warp][lane * V + v] = y[v];
      if (lane == 0) acc[warp][HD] = sum;
      __syncthreads();
      if (warp == 0) {
#pragma unroll
        for (int w = 1; w < W; ++w) {
          sum += acc[w][HD];
#pragma unroll
          for (int v = 0; v < V; ++v) y[v] += acc[w][lane * V + v];
        }
      }
    }
    if (!share || warp == 0) {
      const int flat = st.row0 + row;
      const int64_t node = st.s0 + flat / p.group;
      const int head = st.kvh * p.group + flat % p.group;
#pragma unroll
      for (int v = 0; v < V; ++v) y[v] = sum == 0.f ? 0.f : y[v] / sum;
      uint32_t* out = reinterpret_cast<uint32_t*>(p.out + node * p.out_n + head * p.out_h) + lane * (V / 2);
#pragma unroll
      for (int v = 0; v < V / 2; ++v) out[v] = pack2<DT>(y[2 * v], y[2 * v + 1]);
      if (lane == 0 && p.lse) p.lse[node * p.heads + head] = sum == 0.f ? -INFINITY : (m + log2f(sum)) * 0.6931471805599453f;
    }
  }
}

}  // namespace kv4
}  // namespace af
