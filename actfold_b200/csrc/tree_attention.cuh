// Parts that the two tree attention kernels share: the work list and its
// split over the CTAs, the loads of paged keys and values, small PTX helpers.
#pragma once

#include <cuda.h>

#include <atomic>

#include "tree.cuh"

namespace af {
namespace tree_attn {

constexpr int kKeys = 128;                  // keys per tile
constexpr int kHalf = kKeys * 128;          // [128 rows][64 columns] of 16 bits, 128-byte swizzle
constexpr int kPlans = 4;                   // segments planned in shared memory, up to two ahead of the products of O
// A row of at most this many tiles is not shared by CTAs. Device time with 2 / 4 / 8 / 16 (the results' last bits depend on
// it): one token, 28 heads over 4, 1000 keys 13.5 / 13.4 / 17.1 / 17.0 us; one tree of 26 nodes, the same heads, 900 keys 23.5 /
// 23.5 / 31 / 30.4; 32 requests of 4 nodes over 300 to 4100 keys 46.7 / 46.7 / 55.2 / 62.9; 64 requests of one token over 90 to
// 8000 keys 92.0 / 91.9 / 92.1 / 97.9; 8 trees of 20 to 64 nodes, 32 heads 76.6 / 78.7 / 78.9 / 88. So where rows are few or of
// middling length a lower bound would take up to a quarter less.
constexpr int kWhole = 8;
constexpr float kUnset = -3.0e38f;          // reference maximum of a row that has seen no key
constexpr float kRaise = 8.f;               // log2 headroom before a reference maximum is raised
// A reference maximum is set this far (log2) below the score that it is taken from: probabilities then lie at 2^kLead, and
// below 2^(kLead + kRaise). fp16 is subnormal below 2^-14 and 0 below 2^-25, which a long cache behind one large score would
// lose; 2^15 is still a number of that type, so its steps are 2^-31 of the largest probability. bf16 has fp32's range.
template <int DT>
constexpr float kLead = DT == AF_DTYPE_F16 ? 7.f : 0.f;

struct Params {
  CUtensorMap q, k, v, kc, vc;
  const int *tables, *lengths, *starts;
  const uint32_t* mask;
  int64_t tables_ld, mask_ld;
  int words, batch, total, kv_heads, group, pages, page, box, nt, nt_q;  // nt: nodes of a row tile, nt_q: of one Q box
  int row_cost;  // of a row tile besides its key tiles, in key tiles: its end drains the pipeline
  int64_t capacity;  // tokens that a table row can hold
  float scale;       // times log2(e)
  const char* v_rows;  // the tree's values, for those that are not finite
  int64_t v_n, v_h;
  char* out;
  int64_t out_n, out_h;
  float* lse;
  int heads;
  char* ws;
  unsigned* status;
  int patience;  // attempts of a wait before it gives up
};

// A request's tree and prefix; no cost where there is nothing to do or the values are bad.
struct Request {
  int s0, n, len, pad, kt, qt;
  int row_cost;
  bool bad, narrow;  // narrow: the last row tile has no second Q box, and a wide CTA takes two of its key tiles at a time
  // Units of a row tile and of a head's row tiles (of all heads and requests below 2^31: checked by the host).
  __device__ __forceinline__ int units(bool last) const { return row_cost + (last && narrow ? (kt + 1) / 2 : kt); }
  __device__ __forceinline__ int head_units() const { return (qt - 1) * units(false) + units(true); }
  __device__ __forceinline__ int cost(int kv_heads) const { return kt ? head_units() * kv_heads : 0; }
};

__device__ __forceinline__ Request request(const Params& p, int b) {
  Request r;
  const int s0 = p.starts[b], s1 = p.starts[b + 1];
  r.len = p.lengths[b];
  r.bad = s0 < 0 || s1 < s0 || s1 > p.total || r.len < 0 || r.len > p.capacity || (p.mask && s1 - s0 > 32 * (int64_t)p.words);
  r.s0 = s0;
  r.row_cost = p.row_cost;
  r.n = r.bad ? 0 : s1 - s0;
  r.pad = (r.len + p.box - 1) & -p.box;
  // The same for every row tile, without a mask too: of a long chain's tiles about half are seen by no row of theirs.
  r.kt = r.n ? (r.pad + r.n + kKeys - 1) / kKeys : 0;
  r.qt = r.n <= p.nt ? 1 : (r.n + p.nt - 1) / p.nt;
  r.narrow = p.nt > p.nt_q && r.n - (r.qt - 1) * p.nt <= p.nt_q;
  return r;
}

// The list of rows, each of row_cost units and one per key tile, cut into one share per CTA: the first `more` shares have each + 1.
struct Shares {
  int each, more;
  __device__ __forceinline__ int begin(int i) const { return each * i + min(i, more); }
  __device__ __forceinline__ int owner(int t) const {
    const int big = more * (each + 1);
    return t < big ? t / (each + 1) : more + (t - big) / each;
  }
};

// The tiles [k0, k1) of one row tile that a CTA works on, as one warp plans
// it and the others read it (k1 = 0: the share is done).
struct __align__(16) Segment {
  int s0, n, len, pad;       // the request's nodes, cached keys, and where the tree's keys begin
  int b, kvh, node0, k0;     // request, head, first node of the row tile
  int k1, whole, row_end;    // all tiles of the row?; list index behind its last unit
  int last;                  // the CTA with the row's last tile, where this one begins a row that others go on with
};
struct Walk {
  int t, end, before;  // next unit, end of the share, units of the requests before b
  int b;
};

// The share's next segment. A row of up to kWhole tiles belongs to the CTA
// whose share it begins in.
__device__ __forceinline__ bool next_segment(const Params& p, Walk& w, Segment& s) {
#pragma unroll 1
  while (w.t < w.end) {
    Request r = request(p, w.b);
#pragma unroll 1
    while (w.t >= w.before + r.cost(p.kv_heads)) {
      w.before += r.cost(p.kv_heads);
      r = request(p, ++w.b);
    }
    const int full = r.units(false), rel = w.t - w.before;
    s.kvh = rel / r.head_units();
    const int in_head = rel - s.kvh * r.head_units(), qt = r.qt == 1 ? 0 : min(in_head / full, r.qt - 1);
    const bool last = qt == r.qt - 1;
    const int units = r.units(last), u = in_head - qt * full, step = last && r.narrow ? 2 : 1;
    s.row_end = w.t - u + units;
    s.node0 = qt * p.nt;
    s.s0 = r.s0;
    s.n = r.n;
    s.len = r.len;
    s.pad = r.pad;
    s.b = w.b;
    const int upto = r.kt <= kWhole ? units : min(units, u + (w.end - w.t));
    w.t += upto - u;
    s.k0 = max(0, u - r.row_cost) * step;
    s.k1 = min(r.kt, (upto - r.row_cost) * step);
    if (r.kt <= kWhole ? u > 0 : s.k1 <= s.k0) continue;  // begun by another CTA; no tile in this share
    s.whole = s.k0 == 0 && s.k1 == r.kt;
    return true;
  }
  s.k1 = 0;
  return false;
}

// What CTA c left for k_tree_attention_join: it began a row tile that CTAs
// c + 1 .. last went on with (last = 0: it did not).
struct Started {
  int last, node0, rows, kvh;
};

template <int DT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (DT == AF_DTYPE_BF16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}

template <int DT>
__device__ __forceinline__ uint16_t to_bits(float x) {
  return (uint16_t)pack2<DT>(x, 0.f);
}

__device__ __forceinline__ bool elect_one() {
  int r;
  asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.s32 %0, 1, 0, q;\n\t}" : "=r"(r));
  return r != 0;
}

__device__ __forceinline__ float ex2(float x) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x));
  return e;
}

// Pairs of fp32 values in one register pair (two results per instruction).
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

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

// C consecutive columns of the thread's TMEM lane. Load and wait are one
// statement: nothing that reads the registers can be placed between them.
template <int C>
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t* r) {
  if constexpr (C == 8) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n\ttcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr)
                 : "memory");
  } else if constexpr (C == 16) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\ttcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
                   "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr)
                 : "memory");
  } else {
    static_assert(C == 32, "columns");
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\ttcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
                   "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
                   "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
                   "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(taddr)
                 : "memory");
  }
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}

// Bits of the warp's 32 keys (nodes j0, j0 + 1, ... of the tree) that node i
// sees; a bit outside the tree means nothing.
__device__ __forceinline__ uint32_t seen_bits(const Params& p, int s0, int i, int j0) {
  if (!p.mask) return i < j0 ? 0u : i - j0 >= 31 ? 0xffffffffu : (2u << (i - j0)) - 1u;
  const uint32_t* row = p.mask + (int64_t)(s0 + i) * p.mask_ld;
  const int w = j0 >> 5;  // j0 may be negative: rounds down
  const uint32_t lo = w >= 0 && w < p.words ? row[w] : 0u, hi = w + 1 >= 0 && w + 1 < p.words ? row[w + 1] : 0u;
  return __funnelshift_r(lo, hi, j0 & 31);
}

template <int DT>
__device__ __forceinline__ bool not_finite(uint32_t bits) {
  constexpr uint32_t e = DT == AF_DTYPE_BF16 ? 0x7f80u : 0x7c00u;
  return (bits & e) == e;
}
template <int DT>
__device__ __forceinline__ float from_bits(uint16_t bits) {
  return load_scalar<DT>(reinterpret_cast<const char*>(&bits), 0);
}

// Tiles of a segment that hold values that are not finite: bit i stands for tiles i * 2^shift and on, 2^shift of them, from
// the segment's first.
__device__ __forceinline__ int found_shift(int tiles) { return max(0, 27 - __clz(tiles - 1 | 1)); }

// Calls visit(x, count) for every eight nodes x .. x + count - 1 of such tiles.
template <typename Visit>
__device__ __forceinline__ void for_found(const Segment* plan, const uint32_t* found, Visit visit) {
  const int k0 = plan->k0, tiles = plan->k1 - k0, pad = plan->pad, n = plan->n, shift = found_shift(tiles);
#pragma unroll 1
  for (uint32_t left = *found; left; left &= left - 1) {
    const int first = (__ffs(left) - 1) << shift;
    const int end = min(n, (k0 + min(tiles, first + (1 << shift))) * kKeys - pad);
#pragma unroll 1
    for (int x = max(0, (k0 + first) * kKeys - pad); x < end; x += 8) visit(x, end - x);
  }
}

// The values that are not finite of a segment, added up: of dim d, for each row [col, end) of the tile, at most W, those that it
// sees (narrow kernel); of dims d .. d + 7, those that node i sees (wide kernel). Eight loads at a time serve all of them, and
// only tiles that hold such values are looked through. A prompt of 4000 nodes, 28 heads over 4, with one such value takes 1.4 ms
// (0.6 without; 22 with all nodes looked through); with all of them looked through one after another, once for each value,
// the row ends of 100000 nodes outlasted the waits. (plan: the segment in shared memory, so that the callers hold no registers
// for this.)
template <int DT, int W>
__device__ __noinline__ void set_aside_rows(const Params& p, const Segment* plan, const uint32_t* found, int col, int end, int d, float* sum) {
  const int s0 = plan->s0, node0 = plan->node0;
  const char* at = p.v_rows + (int64_t)s0 * p.v_n + plan->kvh * p.v_h + 2 * d;
#pragma unroll
  for (int e = 0; e < W; ++e) sum[e] = 0.f;
  for_found(plan, found, [&](int x, int count) {
    uint16_t v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = u < count ? *reinterpret_cast<const uint16_t*>(at + (int64_t)(x + u) * p.v_n) : 0;
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (not_finite<DT>(v[u])) {
#pragma unroll 1
        for (int e = 0; e < end - col; ++e)
          if (seen_bits(p, s0, node0 + (col + e) / p.group, x + u) & 1u) sum[e] += from_bits<DT>(v[u]);
      }
  });
}
template <int DT>
__device__ __noinline__ void set_aside_dims(const Params& p, const Segment* plan, const uint32_t* found, int i, int d, float* sum) {
  const int s0 = plan->s0;
  const char* at = p.v_rows + (int64_t)s0 * p.v_n + plan->kvh * p.v_h + 2 * d;
#pragma unroll
  for (int e = 0; e < 8; ++e) sum[e] = 0.f;
  for_found(plan, found, [&](int x, int count) {
    uint4 v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = u < count ? *reinterpret_cast<const uint4*>(at + (int64_t)(x + u) * p.v_n) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const uint32_t w[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
      bool any = false;
#pragma unroll
      for (int e = 0; e < 8; ++e) any |= not_finite<DT>(w[e / 2] >> (16 * (e & 1)));
      if (any && (seen_bits(p, s0, i, x + u) & 1u)) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint16_t b = (uint16_t)(w[e / 2] >> (16 * (e & 1)));
          if (not_finite<DT>(b)) sum[e] += from_bits<DT>(b);
        }
      }
    }
  });
}

// One warp plans: its CTA's share [t, end) of the list, cut into segments.
struct Planner {
  Walk walk;
  Shares shares;
  int made = 0;
  bool more = true;

  __device__ __forceinline__ static int cost_of(const Params& p, int b, bool& disorder) {
    if (b >= p.batch) return 0;
    const Request r = request(p, b);
    disorder |= p.starts[b + 1] < p.starts[b];
    if (r.bad && blockIdx.x == 0 && p.status) atomicOr(p.status, AF_STATUS_BOUNDS);
    return r.cost(p.kv_heads);
  }

  // Two passes over the requests, 32 at a time: the list's length, and the request that the share begins with. Starts out
  // of order anywhere are trees that overlap, whose units nothing bounds: then there is no list.
  __device__ __forceinline__ void begin(const Params& p, int lane) {
    bool disorder = false;
    const int first_cost = cost_of(p, lane, disorder);
    int all = first_cost;
#pragma unroll 4
    for (int b = lane + 32; b < p.batch; b += 32) all += cost_of(p, b, disorder);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
    if (__any_sync(0xffffffffu, disorder)) all = 0;
    shares.each = all / (int)gridDim.x;
    shares.more = all - shares.each * (int)gridDim.x;
    walk.t = shares.begin(blockIdx.x);
    walk.end = shares.begin(blockIdx.x + 1);
    walk.b = walk.before = 0;
    if (walk.t >= walk.end) return;
#pragma unroll 1
    for (int b0 = 0; b0 < p.batch; b0 += 32) {
      int upto = b0 ? cost_of(p, b0 + lane, disorder) : first_cost;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
      }
      const uint32_t behind = __ballot_sync(0xffffffffu, walk.t < walk.before + upto);  // lanes whose request ends behind t
      if (behind) {
        const int x = __ffs(behind) - 1;
        walk.b = b0 + x;
        walk.before += x ? __shfl_sync(0xffffffffu, upto, x - 1) : 0;
        break;
      }
      walk.before += __shfl_sync(0xffffffffu, upto, 31);
    }
  }

  // Publish the segments up to number `upto`.
  __device__ __forceinline__ void on(const Params& p, Segment* plans, uint32_t plan_full, int upto, int lane) {
    Segment s;
#pragma unroll 1
    for (; more && made <= upto; ++made) {
      more = next_segment(p, walk, s);
      s.last = s.k1 > 0 && !s.whole && s.k0 == 0 ? shares.owner(s.row_end - 1) : 0;  // the CTA with the row's last tile
      if (lane == 0) {
        plans[made % kPlans] = s;
        mbar_arrive(plan_full + 8 * (made % kPlans));
      }
      __syncwarp();
    }
  }
};

// Segment number `seg` as it was planned; false behind the last one.
__device__ __forceinline__ bool read_plan(const Segment* plans, uint32_t plan_full, int seg, Segment& s, volatile int* failed) {
  const bool there = __all_sync(0xffffffffu, wait_for(plan_full + 8 * (seg % kPlans), (seg / kPlans) & 1, failed));
  if (!there) *failed = 1;
  s = plans[seg % kPlans];
  return there && s.k1 > 0;
}

// Loads of one operand by a warp: K (with the Q of each segment) or V.
template <typename S, bool VALUES, typename Planned>
__device__ __forceinline__ void load_tiles(const Params& p, Planned planned, uint32_t base, uint32_t full, uint32_t empty, uint32_t q_full,
                                           uint32_t q_empty, volatile int* failed) {
  constexpr int kStages = VALUES ? S::kVStages : S::kKStages;
  const int lane = threadIdx.x & 31;
  const CUtensorMap* cache = VALUES ? &p.vc : &p.kc;
  const CUtensorMap* tree_rows = VALUES ? &p.v : &p.k;
  if (lane < (VALUES ? 2 : 3) && (lane > 0 || p.capacity > 0)) tma_prefetch_desc(lane == 0 ? cache : lane == 1 ? tree_rows : &p.q);
  const int boxes = kKeys / p.box, page_step = kKeys / p.page, off_step = kKeys % p.page;
  int j = 0, seg = 0;
  bool ok = true;
  Segment s;
#pragma unroll 1
  while (ok && planned(seg, s)) {
    const int* table = p.tables + (int64_t)s.b * p.tables_ld;
    // Lane x knows where rows [x * R, (x + 1) * R) of a tile come from (a page is fetched a tile ahead); one lane issues.
    const int row = lane * p.box;
    int key = s.k0 * kKeys + row;
    int entry = key / p.page, off = key - entry * p.page;  // its table entry and place in the page, carried from tile to tile
    int page = lane < boxes && key < s.len ? table[entry] : 0;
    if constexpr (!VALUES) {
      const int qb = seg % S::kQ, use = seg / S::kQ;
      if (use > 0) ok = __all_sync(0xffffffffu, wait_for(q_empty + 8 * qb, (use - 1) & 1, failed));
      if (!ok) break;
      if (elect_one()) {
        const int tiles = s.n - s.node0 > p.nt_q ? S::kQTiles : 1;
        mbar_arrive_expect_tx(q_full + 8 * qb, tiles * S::kHalves * p.nt_q * p.group * 128);
        for (int x = 0; x < tiles * S::kHalves; ++x)
          tma_load_3d(base + S::kOffQ + qb * S::kQBytes + x * S::kQRows * 128, &p.q, q_full + 8 * qb, 64 * (x % S::kHalves), s.kvh * p.group,
                      s.s0 + s.node0 + x / S::kHalves * p.nt_q);
      }
      __syncwarp();
    }
    ++seg;
#pragma unroll 1
    for (int kt = s.k0; kt < s.k1; ++kt, ++j) {
      const int node = key - s.pad;
      const bool cached = lane < boxes && key < s.len, tree = lane < boxes && node >= 0 && node < s.n;
      if (cached && (page < 0 || page >= p.pages)) {
        if (p.status) atomicOr(p.status, AF_STATUS_BOUNDS);
        page = p.pages;  // out of range: the box reads as zeros
      }
      const int from = cached ? off : s.s0 + node, of_page = page;
      const uint32_t from_cache = __ballot_sync(0xffffffffu, cached), from_tree = __ballot_sync(0xffffffffu, tree);
      key += kKeys;
      entry += page_step;
      off += off_step;
      if (off >= p.page) {
        off -= p.page;
        ++entry;
      }
      page = lane < boxes && kt + 1 < s.k1 && key < s.len ? table[entry] : 0;
      const int stage = j % kStages, round = j / kStages;
      if (round > 0) ok = __all_sync(0xffffffffu, wait_for(empty + 8 * stage, (round - 1) & 1, failed));
      if (!ok) break;
      const uint32_t bar = full + 8 * stage;
      const uint32_t dst = base + (VALUES ? S::kOffV : S::kOffK) + stage * S::kStage;
      if (elect_one()) mbar_arrive_expect_tx(bar, __popc(from_cache | from_tree) * p.box * 128 * S::kHalves);
      __syncwarp();
#pragma unroll 1
      for (int x = 0; x < boxes; ++x) {
        const int pg = __shfl_sync(0xffffffffu, of_page, x), at = __shfl_sync(0xffffffffu, from, x);
        const uint32_t to = dst + x * p.box * 128;
        if ((from_cache >> x) & 1u) {
          if (elect_one()) {
            tma_load_4d(to, cache, bar, 0, s.kvh, at, pg);
            if (S::kHalves == 2) tma_load_4d(to + kHalf, cache, bar, 64, s.kvh, at, pg);
          }
        } else if ((from_tree >> x) & 1u) {
          if (elect_one()) {
            tma_load_3d(to, tree_rows, bar, 0, s.kvh, at);
            if (S::kHalves == 2) tma_load_3d(to + kHalf, tree_rows, bar, 64, s.kvh, at);
          }
        }
        __syncwarp();
      }
    }
  }
  if (!ok) {
    *failed = 1;
    if (lane == 0 && p.status) atomicOr(p.status, AF_STATUS_TIMEOUT);
  }
  __syncwarp();
  if (lane == 0) {
    // Copies still in flight (there are some only when a wait ran out, here or in another warp, by now or later) land before
    // the CTA's shared memory is given up (bounded).
    volatile int by_itself[2] = {0, kPatience};
#pragma unroll 1
    for (int i = max(0, j - kStages); i < j; ++i) wait_for(full + 8 * (i % kStages), (i / kStages) & 1, by_itself);
    if (!VALUES)
#pragma unroll 1
      for (int i = max(0, seg - S::kQ); i < seg; ++i) wait_for(q_full + 8 * (i % S::kQ), (i / S::kQ) & 1, by_itself);
  }
  __syncwarp();
}

// After a wait has run out: the products that the two issue warps have in flight end before the CTA's tensor and shared
// memory is given up. Called by both (converged) behind the CTA's last barrier; the one that frees tensor memory waits, for
// both (bounded): a commit follows the products of the thread that makes it.
__device__ __forceinline__ void drain_products(uint32_t drained, bool waits) {
  if (elect_one()) tc_commit(drained);
  __syncwarp();
  volatile int by_itself[2] = {0, kPatience};
  if (waits) wait_for(drained, 0, by_itself);
  __syncwarp();
}

// Workspace: Started[ctas], then per CTA two partial rows (0: begun by an
// earlier CTA, 1: begun here) of [N][HD] fp32 sums and [N] (maximum, sum) pairs.
template <int N, int HD>
struct Scratch {
  char* base;
  int ctas;
  __host__ __device__ static int64_t bytes(int ctas) { return ctas * (int64_t)(sizeof(Started) + 2 * N * (HD + 2) * 4); }
  __device__ Started* started(int c) const { return reinterpret_cast<Started*>(base) + c; }
  __device__ float* sums(int c, int which) const {
    return reinterpret_cast<float*>(base + ctas * sizeof(Started)) + ((int64_t)c * 2 + which) * N * HD;
  }
  __device__ float2* stats(int c, int which) const {
    return reinterpret_cast<float2*>(base + ctas * (sizeof(Started) + (int64_t)2 * N * HD * 4)) + ((int64_t)c * 2 + which) * N;
  }
};

// The wide kernel (tree_attention_wide.cu) and the joins of shared rows.
int wide_launch(const Params& p, bool bf16, int head_dim, cudaStream_t s);
template <int DT, int N, int HD>
int join_launch(const Params& p, int ctas, cudaStream_t s);

// Let a kernel use this much shared memory, once per device.
template <auto Kernel>
int allow_smem(int bytes) {
  static std::atomic<uint64_t> allowed{0};  // a bit per device
  int device = 0;
  cudaGetDevice(&device);
  const uint64_t bit = 1ull << (device & 63);
  if (allowed.load(std::memory_order_relaxed) & bit) return AF_OK;
  const cudaError_t e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return fail(AF_ERR_CUDA, std::string("af_tree_attention: ") + cudaGetErrorString(e));
  allowed.fetch_or(bit, std::memory_order_relaxed);
  return AF_OK;
}

}  // namespace tree_attn
}  // namespace af
