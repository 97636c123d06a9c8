// Attention over the 4-bit paged cache with many rows per key/value head
// (sm_100a, tcgen05): the list of work and the joins of int4_attention.cuh, but the
// rows are the M side (S [128 rows, 128 keys] = Q K^T, O += P V), because with
// more than 16 rows a tile of keys is worth turning into 16 bits once, in
// shared memory, for all rows.
//
// A CTA holds two "pipes", each a 128-row O and a 128-row S of 128 keys, over
// which P is written in place (16 bits, TMEM operand of the second product).
// With more than 128 rows they are two row tiles over the same keys; with
// fewer, one row tile over the even and the odd key tiles, joined at the end.
// Four warps turn a tile's keys into values and write them where the tensor cores take
// them (a thread has a key; 16-byte pieces, 128-byte swizzle), four others the values; the next tile's codes are brought into the L2
// meanwhile. A softmax thread owns a row, so no scores are exchanged. The reference maximum of a row is raised only when a
// score passes it by 2^8.
//
// Probabilities are rounded to the values' type as in int4_attention.cu: half a step of each, in the place of S.
//
// The work of a tile: 64 KB that go through shared memory twice (some 1000 cycles of its 128 bytes), 512 cycles of products per
// pipe, 128 exponentials a row. No unit is busy all the time: it is the chain of turning, product, softmax and product, through
// two buffers, that bounds it (per tile some 5500 cycles with one row tile, of which the turning warps take some 4300 with what they wait for; the softmax
// 1500 to 1900 for half a tile of 128 rows).
//   8 trees of 20 to 64 nodes, 32 heads over 32, 300 to 4100 keys: 246 us with the kernel of few rows, 94 now; its bytes need 17.
//   4 trees of 48 to 64 nodes, 28 heads over 4, 30 to 65 K keys: 2204 us with that kernel, 259 now; its products need 107.
// (The 16-bit cache's attention takes 79 and 252 to 257 us for them: the codes' turning costs what their fewer bytes gain.)
// Tried: keys and values one after the other in eight warps (114 us instead of 105 at that time: a tile's keys waited for the
// products with the values two tiles before); 16 turning warps with 72 registers, more registers for the issue warps or the turning
// ones, the codes a tile ahead in shared memory (the long trees 259 -> 274 us) or half a tile ahead in registers (the first 93 -> 105), halves of S
// with one row tile too (96 -> 99): slower.
//
// Warps 0-3 and 4-7: softmax of pipe 0 and 1, and Q; 8-11: keys; 12-15: values; 16 issues S, 17 O, 18 plans, 19 is idle.
#include "int4_attention.cuh"

namespace af {
namespace kv4 {

namespace {

constexpr int kUnit = kWideUnit;           // keys of a tile
constexpr int kRows = 128;                 // rows of a pipe
constexpr int kSoft = 8, kTurn = 8;         // warps for the softmax; for keys and values, half of them each
constexpr int kMmaS = kSoft + kTurn, kMmaO = kMmaS + 1, kPlan = kMmaS + 2;
constexpr int kThreads = 32 * (kPlan + 2);  // (whole groups of four warps share out registers)
constexpr int kReaders = kSoft + kTurn + 2;  // of a plan
constexpr int kStages = 2;                 // of keys, and of values
constexpr int kPanel = kUnit * 128;        // [128 rows][64 columns] of 16 bits, 128-byte swizzle

template <int HD>
struct Wide {
  static constexpr int kHalves = HD / 64;
  static constexpr int kTile = kHalves * kPanel;  // a K, V or Q tile
  static constexpr int kOffK = 0, kOffV = kStages * kTile, kOffQ = 2 * kStages * kTile;
  static constexpr int kOffStat = kOffQ + 2 * kTile;                 // [2][128] (maximum, sum) of the pipes
  static constexpr int kOffBar = kOffStat + 2 * kRows * 8;
  static constexpr int kBars = 4 * kStages + 1 + 12 + 2 + 2 * kPlans + 1;
  static constexpr int kOffPlan = (kOffBar + 8 * kBars + 15) / 16 * 16;
  static constexpr int kOffMisc = kOffPlan + kPlans * (int)sizeof(Segment);  // tensor memory's address; failed, patience; found[kPlans]
  static constexpr int kBytes = kOffMisc + 4 * (4 + kPlans);
  static constexpr int kTmemO = 2 * kUnit;                           // O of pipe x at kTmemO + 128 x, S of pipe x at 128 x
};

__device__ __forceinline__ bool elect_one() {
  int r;
  asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.s32 %0, 1, 0, q;\n\t}" : "=r"(r));
  return r != 0;
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

// C consecutive columns of the thread's TMEM lane. Load and wait are one
// statement: nothing that reads the registers can be placed between them.
__device__ __forceinline__ void tmem_load8(uint32_t taddr, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n\ttcgen05.wait::ld.sync.aligned;"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_load16x2(uint32_t a, uint32_t b, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%32];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%33];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
        "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
        "=r"(r[31])
      : "r"(a), "r"(b)
      : "memory");
}
__device__ __forceinline__ void tmem_store8(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
// 64 consecutive columns of the thread's TMEM lane.
__device__ __forceinline__ void tmem_load64(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%64];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%65];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]), "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]), "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
      : "r"(taddr), "r"(taddr + 32)
      : "memory");
}

__device__ __forceinline__ void tmem_store32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

__device__ __forceinline__ void tmem_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// D [tmem] (+)= A [smem] * B [smem]^T.
__device__ __forceinline__ void mma_from_smem(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// D [tmem] (+)= A [tmem, 16-bit pairs] * B [smem]^T.
__device__ __forceinline__ void mma_from_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ uint32_t below(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }

// Place of unit x of a segment's cached keys.
__device__ __forceinline__ int place_of(const Segment& s, int x) { return kUnit * (x < s.sink_units ? x : x - s.sink_units + s.from); }

// Not every row of the request sees all of these keys: the prefix's last ones, ones that only some windows hold, and nodes.
__device__ __forceinline__ bool is_masked(const Params& p, const Segment& s, int x) {
  if (x >= s.cached) return true;
  const int place = place_of(s, x);
  return place + kUnit > s.len || (p.window && place < s.len - max(0, p.window - s.n) && place + kUnit > p.sinks);
}

// Units of a segment that hold values that are not finite and that not all rows see: bit i stands for units i * 2^shift and on,
// 2^shift of them, from the segment's first.
__device__ __forceinline__ int found_shift(int units) { return max(0, 27 - __clz(units - 1 | 1)); }

// Such values of dims d .. d + 15, added up for a row of node i, whose window begins at `first`. (Four keys' loads at a time: of a
// long chain with such values in every unit a row's end looks through all nodes.)
template <int DT, int HD>
__device__ __noinline__ void set_aside(const Params& p, const Segment* plan, uint32_t found, int i, int first, int d, float* sum) {
  using B = Block<HD>;
  const Segment& s = *plan;
  const int units = s.x1 - s.x0, shift = found_shift(units);
#pragma unroll
  for (int e = 0; e < 16; ++e) sum[e] = 0.f;
#pragma unroll 1
  for (; found; found &= found - 1) {
    const int u0 = (__ffs(found) - 1) << shift;
#pragma unroll 1
    for (int x = s.x0 + u0; x < s.x0 + min(units, u0 + (1 << shift)); ++x) {
      if (!is_masked(p, s, x)) continue;
      if (x < s.cached) {
        const int place0 = place_of(s, x), end = min(s.len, place0 + kUnit);
        bool bad = false;
#pragma unroll 4
        for (int at = place0; at < end; ++at) {
          const int entry = entry_of(p, at), off = at - entry * p.page, page = p.tables[(int64_t)s.b * p.tables_ld + entry];
          uint32_t pr = 0;
          if ((at >= first || at < p.sinks) && page >= 0 && page < p.pages)
            pr = *reinterpret_cast<const uint32_t*>(p.data + page * p.d_page + s.kvh * p.d_head + (int64_t)(off / kBlockTokens) * B::kBytes + B::kPart +
                                                    B::pair(off % kBlockTokens, d / kGroup));
          bad |= not_finite<DT>(pr) || not_finite<DT>(pr >> 16);
        }
        if (bad)
#pragma unroll
          for (int e = 0; e < 16; ++e) sum[e] = NAN;
      } else {
        const int n0 = kUnit * (x - s.cached), end = min(s.n, n0 + kUnit);
        const char* from = p.v + (int64_t)s.s0 * p.v_n + s.kvh * p.v_h + 2 * d;
#pragma unroll 1
        for (int j = n0; j < end; j += 4) {
          uint4 v[4][2];
#pragma unroll
          for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              v[u][h] = j + u < end ? *reinterpret_cast<const uint4*>(from + (int64_t)(j + u) * p.v_n + 16 * h) : make_uint4(0, 0, 0, 0);
          const uint32_t seen = seen_nodes(p, s.s0, s.n, s.len, i, j & ~31) >> (j & 31);
#pragma unroll
          for (int u = 0; u < 4; ++u)
            if ((seen >> u) & 1u) {
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                const uint32_t w = reinterpret_cast<const uint32_t*>(&v[u][e / 8])[e % 8 / 2], b = (w >> (16 * (e & 1))) & 0xffffu;
                if (not_finite<DT>(b)) sum[e] += from_bits<DT>(b);
              }
            }
        }
      }
    }
  }
}

template <int R>
__device__ __forceinline__ void registers_up() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R));
}
template <int R>
__device__ __forceinline__ void registers_down() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R));
}
constexpr int kRegsSoft = 152, kRegsTurn = 64, kRegsRest = 48;  // of a thread; at launch all have 96
static_assert(kThreads == 20 * 32 && 8 * kRegsSoft + 8 * kRegsTurn + 4 * kRegsRest <= 20 * 96, "no more than the launch has");

template <int DT, int HD>
__global__ void __launch_bounds__(kThreads, 1) k_int4_attention_wide(const __grid_constant__ Params p) {
  using S = Wide<HD>;
  using B = Block<HD>;
  extern __shared__ __align__(1024) uint8_t gb[];
  pdl_trigger();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t base = smem_u32(gb);
  const uint32_t k_full = base + S::kOffBar, k_empty = k_full + 8 * kStages, v_full = k_empty + 8 * kStages, v_empty = v_full + 8 * kStages,
                 q_full = v_empty + 8 * kStages, s_full = q_full + 8, p_full = s_full + 32, done = p_full + 32, o_full = done + 32, o_empty = o_full + 8,
                 plan_full = o_empty + 8, plan_empty = plan_full + 8 * kPlans, drained = plan_empty + 8 * kPlans;
  Segment* plans = reinterpret_cast<Segment*>(gb + S::kOffPlan);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(gb + S::kOffMisc);
  volatile int* failed = reinterpret_cast<volatile int*>(tmem_slot + 1);
  uint32_t* found = tmem_slot + 4;  // per plan: units with values that are not finite

  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(k_full + 8 * i, 4);
      mbar_init(k_empty + 8 * i, 1);
      mbar_init(v_full + 8 * i, 4);
      mbar_init(v_empty + 8 * i, 1);
    }
    for (int i = 0; i < 4; ++i) {  // [pipe][half]
      mbar_init(s_full + 8 * i, 1);
      mbar_init(p_full + 8 * i, 4);
      mbar_init(done + 8 * i, 1);
    }
    mbar_init(q_full, kSoft);
    mbar_init(o_full, 1);
    mbar_init(o_empty, kSoft);
    for (int i = 0; i < kPlans; ++i) {
      mbar_init(plan_full + 8 * i, 1);
      mbar_init(plan_empty + 8 * i, kReaders);
    }
    mbar_init(drained, 2);
    failed[0] = 0;
    failed[1] = p.patience;
    fence_barrier_init();
  }
  if (warp == kMmaS) tmem_alloc(smem_u32(tmem_slot), 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const Scratch<2 * kRows, HD> scratch{p.ws, (int)gridDim.x};
  Segment s;
  auto agreed = [](bool mine) { return (bool)__all_sync(0xffffffffu, mine); };
  // Segment number `seg` as it was planned; false behind the last one. Its reader gives it back with read().
  auto planned = [&](int seg, Segment& s) {
    const bool there = agreed(wait_for(plan_full + 8 * (seg % kPlans), (seg / kPlans) & 1, failed));
    if (!there) *failed = 1;
    s = plans[seg % kPlans];
    return there && s.x1 > 0;
  };
  auto read = [&](int seg) {
    __syncwarp();
    if (lane == 0) mbar_arrive(plan_empty + 8 * (seg % kPlans));
  };
  auto give_up = [&]() {
    *failed = 1;
    if (lane == 0 && p.status) atomicOr(p.status, AF_STATUS_TIMEOUT);
  };
  constexpr uint32_t kind = DT == AF_DTYPE_BF16 ? 0u : ((1u << 7) | (1u << 10));  // operand formats: bf16 = 1, f16 = 0

  if (warp >= kMmaS) registers_down<kRegsRest>();
  if (warp == kPlan) {
    Planner<kUnit> planner;
    planner.begin(p, lane);
    bool ok = true;
#pragma unroll 1
    for (int seg = 0; ok; ++seg) {
      const bool more = planner.next(p, s);
      if (seg >= kPlans) ok = agreed(wait_for(plan_empty + 8 * (seg % kPlans), (seg / kPlans - 1) & 1, failed));
      if (!ok) break;
      if (lane == 0) {
        plans[seg % kPlans] = s;
        found[seg % kPlans] = 0;
        mbar_arrive(plan_full + 8 * (seg % kPlans));
      }
      __syncwarp();
      if (!more) break;
    }
    if (!ok) give_up();
  } else if (warp == kMmaS) {
    // ---------------- S: two row tiles of a key tile, or one of every other key tile ----------------
    // With two, 64 keys at a time: a half's S goes where P of the half before it has been multiplied, while the softmax works on
    // the other half (4 requests of 64 nodes x 7 heads over up to 65 K keys 268 -> 255 us). With one the other pipe fills the gaps,
    // and products of 64 columns cost three quarters of those of 128 (8 trees of 20 to 64 nodes, 32 heads 96 -> 99 us).
    constexpr uint32_t id_half = idesc_bf16(kRows, kUnit / 2) ^ kind, id_all = idesc_bf16(kRows, kUnit) ^ kind;
    const uint64_t d_k = sw128_desc(base + S::kOffK), d_q = sw128_desc(base + S::kOffQ);
    bool ok = true;
    int seg = 0, j = 0, used0 = 0, used1 = 0;  // tiles; tiles of S of the pipes
#pragma unroll 1
    while (ok && planned(seg, s)) {
      const bool two = s.n * p.group - s.row0 > kRows && p.rows > kRows;
      const int tiles = s.x1 - s.x0, steps = two ? 4 : 1;  // of a key tile
      ok = agreed(wait_for(q_full, seg & 1, failed));
#pragma unroll 1
      for (int t = 0; ok && t < tiles; ++t, ++j) {
        const int stage = j % kStages;
        ok = agreed(wait_for(k_full + 8 * stage, (j / kStages) & 1, failed));
#pragma unroll 1
        for (int x = 0; ok && x < steps; ++x) {
          const int half = two ? x >> 1 : 0, pipe = two ? x & 1 : t & 1, bar = 2 * pipe + half, used = pipe ? used1 : used0;
          if (used) ok = agreed(wait_for(done + 8 * (two ? bar : bar + 1), (used - 1) & 1, failed));  // P V of the last keys there
          if (!ok) break;
          tc_fence_after();
          const uint64_t a = d_q + ((p.rows > kRows ? two && pipe : seg & 1) ? (uint32_t)S::kTile >> 4 : 0u), b = d_k + (uint32_t)stage * (S::kTile >> 4) + half * (kPanel >> 5);
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < HD / 16; ++kk)
              mma_from_smem(tmem + 128 * pipe + 64 * half, a + (kk >> 2) * (kPanel >> 4) + 2 * (kk & 3), b + (kk >> 2) * (kPanel >> 4) + 2 * (kk & 3),
                            two ? id_half : id_all, kk ? 1u : 0u);
            tc_commit(s_full + 8 * bar);
            if (!two) tc_commit(s_full + 8 * (bar + 1));
            if (x == steps - 1) tc_commit(k_empty + 8 * stage);
          }
          __syncwarp();
        }
        used0 += two || !(t & 1);
        used1 += two || (t & 1);
      }
      read(seg++);
    }
    if (!ok) give_up();
  } else if (warp == kMmaO) {
    // ---------------- O += P V of every half ----------------
    constexpr uint32_t id_o = idesc_bf16_bmn(kRows, HD) ^ kind;
    const uint64_t d_v = sw128_desc_mn(base + S::kOffV, kPanel, 1024);
    bool ok = true;
    int seg = 0, j = 0, used0 = 0, used1 = 0;
#pragma unroll 1
    while (ok && planned(seg, s)) {
      const bool two = s.n * p.group - s.row0 > kRows && p.rows > kRows;
      const int tiles = s.x1 - s.x0, steps = two ? 4 : 2;
      if (seg > 0) ok = agreed(wait_for(o_empty, (seg - 1) & 1, failed));  // the last segment's O is read
#pragma unroll 1
      for (int t = 0; ok && t < tiles; ++t, ++j) {
        const int stage = j % kStages, x1 = s.x0 + t;
        ok = agreed(wait_for(v_full + 8 * stage, (j / kStages) & 1, failed));
        const int keys16 = ((x1 < s.cached ? s.len - place_of(s, x1) : s.n - kUnit * (x1 - s.cached)) + 15) / 16;  // up to the tile's last key
#pragma unroll 1
        for (int x = 0; ok && x < steps; ++x) {
          const int half = two ? x >> 1 : x, pipe = two ? x & 1 : t & 1, bar = 2 * pipe + half, used = pipe ? used1 : used0;
          ok = agreed(wait_for(p_full + 8 * bar, used & 1, failed));
          if (!ok) break;
          tc_fence_after();
          const uint64_t b = d_v + (uint32_t)stage * (S::kTile >> 4) + half * 4 * 128;
          const uint32_t o = tmem + S::kTmemO + 128 * pipe, a = tmem + 128 * pipe + 64 * half;
          const uint32_t add = t > (two ? 0 : 1) || half;
          const int keys = keys16 - 4 * half;
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              if (kk < keys) mma_from_tmem(o, a + 8 * kk, b + kk * 128, id_o, kk ? 1u : add);
            tc_commit(done + 8 * bar);
            if (x == steps - 1) tc_commit(v_empty + 8 * stage);
            if (x == steps - 1 && t == tiles - 1) tc_commit(o_full);
          }
          __syncwarp();
        }
        used0 += two || !(t & 1);
        used1 += two || (t & 1);
      }
      read(seg++);
    }
    if (!ok) give_up();
  } else if (warp >= kSoft && warp < kMmaS) {
    registers_down<kRegsTurn>();
    // ---------------- keys or values into 16 bits: thread = a key of every tile ----------------
    constexpr int kWords = HD / 8, kPairs = HD / 32;
    const bool values = warp >= kSoft + kTurn / 2;
    const int key = tid & 127;
    const uint32_t full = values ? v_full : k_full, empty = values ? v_empty : k_empty;
    const uint32_t tiles_at = base + (values ? S::kOffV : S::kOffK) + key * 128;
    auto write = [&](uint32_t tile, int i, uint4 v) {  // dims 8 i .. 8 i + 7
      asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(tile + (i >> 3) * kPanel + 16 * ((i & 7) ^ (key & 7))), "r"(v.x), "r"(v.y), "r"(v.z),
                   "r"(v.w)
                   : "memory");
    };
    // The next tile: unit x of segment seg, its place of the thread's key (-1: none that is cached) and that one's page.
    int seg = 0, x = 0, at = -1, page = 0;
    auto look_up = [&]() {
      const Segment& f = plans[seg % kPlans];
      at = x < f.cached ? place_of(f, x) + key : f.len;
      if (at >= f.len) at = -1;
      page = at < 0 ? 0 : p.tables[(int64_t)f.b * p.tables_ld + entry_of(p, at)];
    };
    auto begin = [&]() {  // unit 0 of segment seg
      if (!agreed(wait_for(plan_full + 8 * (seg % kPlans), (seg / kPlans) & 1, failed))) {
        *failed = 1;
        return false;
      }
      x = plans[seg % kPlans].x0;
      return plans[seg % kPlans].x1 > 0;
    };
    uint32_t w[kWords], pr[kPairs];
    // Where the thread's codes and pairs lie: they are brought into the L2 while the tile before is worked on. Null where there is no
    // cached key, and of a page out of range.
    const int r = key % kBlockTokens;  // (units begin with a block)
    const char* from = nullptr;
    auto locate = [&]() {
      from = nullptr;
      if (at < 0) return;
      if (page < 0 || page >= p.pages) {
        if (p.status) atomicOr(p.status, AF_STATUS_BOUNDS);
        return;
      }
      const int off = at - entry_of(p, at) * p.page;
      from = p.data + page * p.d_page + plans[seg % kPlans].kvh * p.d_head + (off / kBlockTokens) * B::kBytes + (values ? B::kPart : 0);
      prefetch_l2(from + B::word(r, 0));
      prefetch_l2(from + B::pair(r, 0));
    };
    // They; zeros where there are none.
    auto fetch = [&]() {
#pragma unroll
      for (int i = 0; i < kWords; ++i) w[i] = 0;
#pragma unroll
      for (int i = 0; i < kPairs; ++i) pr[i] = 0;
      if (!from) return;
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i) {
        const uint4 y = *reinterpret_cast<const uint4*>(from + B::word(r, 4 * i));
        w[4 * i] = y.x, w[4 * i + 1] = y.y, w[4 * i + 2] = y.z, w[4 * i + 3] = y.w;
      }
      if constexpr (HD == 128) {
        const uint4 y = *reinterpret_cast<const uint4*>(from + B::pair(r, 0));
        pr[0] = y.x, pr[1] = y.y, pr[2] = y.z, pr[3] = y.w;
      } else {
        const uint2 y = *reinterpret_cast<const uint2*>(from + B::pair(r, 0));
        pr[0] = y.x, pr[1] = y.y;
      }
    };
    bool ok = true, more = begin();
    if (more) {
      look_up();
      locate();
      fetch();
    }
    int done_with = 0;  // segments that this warp no longer reads
#pragma unroll 1
    while (more) {
      const Segment& f = plans[seg % kPlans];
      const int now = seg, x_now = x, at_now = at, j = f.j0 + x - f.x0, stage = j % kStages;
      const uint32_t tile = tiles_at + stage * S::kTile;
      const bool cached = x < f.cached;
      // The next tile's page is looked up meanwhile. (Each segment has a tile: the next lies at most one segment on, which is planned
      // while this one is still held.)
      more = ++x < f.x1;
      if (!more) {
        ++seg;
        more = begin();
      }
      if (more) look_up();
      bool sick = false;
      if (values && cached && is_masked(p, f, x_now)) {
        // What no row sees is 0 (as what there is no key for); NaN that only some rows see is set aside.
        const bool hidden = at_now < 0 || (p.window && at_now < f.len - p.reach && at_now >= p.sinks);
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
          if (hidden) pr[i] = 0;
          if (not_finite<DT>(pr[i]) || not_finite<DT>(pr[i] >> 16)) {
            sick = true;
            pr[i] = 0;
          }
        }
      }
      if (j >= kStages) ok = agreed(wait_for(empty + 8 * stage, (j / kStages - 1) & 1, failed));
      if (!ok) break;
      if (more) locate();
      if (cached) {
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
          const uint32_t s2 = __byte_perm(pr[i / 4], 0, 0x1010), o2 = __byte_perm(pr[i / 4], 0, 0x3232);
          write(tile, i, make_uint4(two_values<DT, 0>(w[i], s2, o2), two_values<DT, 1>(w[i], s2, o2), two_values<DT, 2>(w[i], s2, o2),
                                    two_values<DT, 3>(w[i], s2, o2)));
        }
      } else {
        // A node's row, zeros behind the last node; of values the ones that are not finite are set aside.
        const int node = kUnit * (x_now - f.cached) + key;
        const char* row = values ? p.v + (int64_t)(f.s0 + node) * p.v_n + f.kvh * p.v_h : p.k + (int64_t)(f.s0 + node) * p.k_n + f.kvh * p.k_h;
        const bool there = node < f.n;
#pragma unroll 4
        for (int i = 0; i < kWords; ++i) {
          uint4 v = there ? *reinterpret_cast<const uint4*>(row + 16 * i) : make_uint4(0, 0, 0, 0);
          if (values) {
            uint32_t* y = &v.x;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const bool lo = not_finite<DT>(y[e]), hi = not_finite<DT>(y[e] >> 16);
              sick |= lo || hi;
              y[e] &= (lo ? 0u : 0xffffu) | (hi ? 0u : 0xffff0000u);
            }
          }
          write(tile, i, v);
        }
      }
      if (sick) atomicOr(&found[now % kPlans], 1u << ((x_now - f.x0) >> found_shift(f.x1 - f.x0)));
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(full + 8 * stage);
      if (more) fetch();  // (on its way while the stage is waited for)
      for (; done_with < seg; ++done_with) read(done_with);
    }
    if (!ok) give_up();
  } else if (warp < kSoft) {
    registers_up<kRegsSoft>();
    // ---------------- softmax of row r of the pipe's tiles ----------------
    const int quad = warp & 3, pipe = warp >> 2, r = 32 * quad + lane;
    const uint32_t lanes = tmem + ((uint32_t)(32 * quad) << 16);
    const uint32_t at_s = lanes + 128 * pipe, at_o = lanes + S::kTmemO + 128 * pipe;
    float2* stat = reinterpret_cast<float2*>(gb + S::kOffStat);
    const float sc = p.scale;
    auto wait = [&](uint32_t bar, uint32_t parity) {
      if (!wait_for(bar, parity, failed)) *failed = 1;
    };
    int seg = 0, taken = 0;  // halves of S of this pipe so far
    bool wrote_start = false;
    // Q of a segment: the thread's row, 16-byte pieces swizzled over 128 bytes; zeros where there is no row. Two row tiles have a
    // buffer each and come when the segment begins, one has both by turns and comes while the one before it is worked on.
    auto q_tile = [&](int number, int pipe) { return p.rows > kRows ? pipe : number & 1; };
    auto bring_q = [&](int number) {
      if (!agreed(wait_for(plan_full + 8 * (number % kPlans), (number / kPlans) & 1, failed))) return;
      const Segment& f = plans[number % kPlans];
      if (f.x1 <= 0) return;
      const int all = min(p.rows, f.n * p.group - f.row0), row = p.rows > kRows ? kRows * pipe + r : r;
      if (p.rows <= kRows ? pipe > 0 : all <= kRows * pipe) return;
      const int flat = f.row0 + min(row, all - 1);
      const char* from = p.q + (int64_t)(f.s0 + flat / p.group) * p.q_n + (f.kvh * p.group + flat % p.group) * p.q_h;
      const uint32_t to = base + S::kOffQ + q_tile(number, pipe) * S::kTile + r * 128;
#pragma unroll
      for (int i = 0; i < HD / 8; ++i)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + (i >> 3) * kPanel + 16 * ((i & 7) ^ (r & 7))), "l"(from + 16 * i),
                     "r"(row < all ? 16 : 0)
                     : "memory");
    };
    // Q of a segment has landed: S may read it.
    auto landed = [&](int number) {
      asm volatile("cp.async.wait_all;" ::: "memory");
      if (p.q_flip | ~p.q_keep) {  // (a scale that is not positive)
        const uint32_t mine = base + S::kOffQ + q_tile(number, pipe) * S::kTile + r * 128;
#pragma unroll 1
        for (int i = 0; i < HD / 8 && (p.rows > kRows || pipe == 0); ++i) {
          uint4 v;
          const uint32_t at = mine + (i >> 3) * kPanel + 16 * (i & 7);
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"((v.x ^ p.q_flip) & p.q_keep), "r"((v.y ^ p.q_flip) & p.q_keep),
                       "r"((v.z ^ p.q_flip) & p.q_keep), "r"((v.w ^ p.q_flip) & p.q_keep)
                       : "memory");
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
    };
    if (p.rows <= kRows) {
      bring_q(0);
      landed(0);
    }
    // Into the next segment go all softmax warps or none, whatever each has seen of a plan or of a wait that ran out: the
    // barriers inside have no limit of their own.
    auto enter = [&]() {
      const bool there = planned(seg, s);
      return !vote_any<kSoft * 32>(1, !there || *failed);
    };
#pragma unroll 1
    while (enter()) {
      const int all = min(p.rows, s.n * p.group - s.row0);   // rows of the tile
      const bool two = all > kRows;
      const int tiles = s.x1 - s.x0;
      const int row = (two && pipe ? kRows : 0) + r;          // of the tile
      const int rows = min(kRows, two && pipe ? all - kRows : all);
      const int flat = s.row0 + min(row, all - 1), node = flat / p.group, head = s.kvh * p.group + flat % p.group;
      const bool busy = 32 * quad < rows;                     // any of the warp's rows is one
      if (p.rows > kRows) bring_q(seg);  // (S of the segment before is complete: all pipes have read it)
      if (p.rows > kRows) landed(seg);
      if (p.rows <= kRows) bring_q(seg + 1);
      const int first = first_place(p, s.s0, s.n, s.len, node);
      float m = kUnset;
      uint64_t l0 = 0ull, l1 = 0ull;
#pragma unroll 1
      for (int x2 = two ? 0 : 2 * pipe; x2 < 2 * tiles; x2 += two || !(x2 & 1) ? 1 : 3, ++taken) {
        const int x = s.x0 + (x2 >> 1), half = x2 & 1, bar = 2 * pipe + half;  // a half of a tile at a time
        const bool cached = x < s.cached, masked = is_masked(p, s, x);
        const int key0 = (cached ? place_of(s, x) : kUnit * (x - s.cached)) + 64 * half;
        wait(s_full + 8 * bar, (taken >> 1) & 1);
        tc_fence_after();
        if (busy) {
          uint32_t vis[2] = {0xffffffffu, 0xffffffffu};
          if (masked) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const int k = key0 + 32 * c;
              if (cached) vis[c] = below(s.len - k) & (~below(first - k) | below(p.sinks - k));
              else vis[c] = r < rows && k < s.n ? seen_nodes(p, s.s0, s.n, s.len, node, k) : 0u;
            }
          }
          constexpr int C = kUnit / 2;
          uint32_t y[C];
          tmem_load64(at_s + C * half, y);
          if (masked) {  // hidden scores are -inf
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (!((vis[c] >> i) & 1u)) y[32 * c + i] = 0xff800000u;
          }
          float top[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            top[c] = __uint_as_float(y[16 * c]);
#pragma unroll
            for (int i = 1; i < 15; i += 2) top[c] = fmaxf(top[c], fmaxf(__uint_as_float(y[16 * c + i]), __uint_as_float(y[16 * c + i + 1])));
            top[c] = fmaxf(top[c], __uint_as_float(y[16 * c + 15]));
          }
          const float t_max = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * sc;
          const bool raise = m == kUnset ? t_max > kUnset : t_max > m + (kLead<DT> + kRaise);
          if (__any_sync(0xffffffffu, raise)) {
            const float f = raise ? (m == kUnset ? 0.f : exp2f(m - (t_max - kLead<DT>))) : 1.f;
            if (raise) m = t_max - kLead<DT>;
            if (x2 > (two ? 0 : 2 * pipe)) {
              // O of the halves before this one is complete once the last one's P V is.
              wait(done + 8 * (bar ^ 1), ((taken - 1) >> 1) & 1);
              tc_fence_after();
              l0 = fma2(l0, pair(f, f), 0ull);
              l1 = fma2(l1, pair(f, f), 0ull);
#pragma unroll 1
              for (int c = 0; c < HD; c += 8) {
                uint32_t o[8];
                tmem_load8(at_o + c, o);
#pragma unroll
                for (int i = 0; i < 8; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                tmem_store8(at_o + c, o);
              }
            }
          }
          const uint64_t sc2 = pair(sc, sc), nm2 = pair(-m, -m);
          uint32_t e[C / 2];
#pragma unroll
          for (int i = 0; i < C / 2; i += 2) {
            const float2 a = unpair(fma2(pair(__uint_as_float(y[2 * i]), __uint_as_float(y[2 * i + 1])), sc2, nm2));
            const float2 b = unpair(fma2(pair(__uint_as_float(y[2 * i + 2]), __uint_as_float(y[2 * i + 3])), sc2, nm2));
            const float a0 = ex2(a.x), a1 = ex2(a.y), b0 = ex2(b.x), b1 = ex2(b.y);
            l0 = add2(l0, pair(a0, a1));
            l1 = add2(l1, pair(b0, b1));
            e[i] = pack2<DT>(a0, a1);
            e[i + 1] = pack2<DT>(b0, b1);
          }
          tmem_store32(at_s + C * half, e);
          tmem_wait_store();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full + 8 * bar);
      }
      if (p.rows <= kRows) landed(seg + 1);  // (its first S are made while this segment's rows are written)
      // ---- the segment's rows ----
      const float2 la = unpair(add2(l0, l1));
      const float mine = la.x + la.y;
      stat[pipe * kRows + r] = make_float2(m, mine);
      named_bar_sync(1, kSoft * 32);
      float own = 1.f, other = 0.f, sum = mine;  // factors of this pipe's O and of the other one's
      if (!two) {
        const float2 y = stat[(1 - pipe) * kRows + r];
        const float top = fmaxf(m, y.x);
        own = m == top ? 1.f : exp2f(m - top);
        other = y.x == top ? 1.f : exp2f(y.x - top);
        // (the same operations in the same order on both sides)
        sum = pipe ? other * y.y + own * mine : own * mine + other * y.y;
        m = top;
      }
      const bool whole = s.whole != 0;
      const int which = s.x0 == 0 ? 1 : 0;
      const float inv = !whole ? 1.f : sum == 0.f ? 0.f : 1.f / sum;
      own *= inv;
      other *= inv;
      const bool single = two || tiles == 1;  // only one pipe's O holds anything of these rows
      wait(o_full, seg & 1);
      tc_fence_after();
      const uint32_t aside = found[seg % kPlans];
      const int d0 = two ? 0 : pipe * (HD / 2), d1 = two ? HD : d0 + HD / 2;  // the columns that this thread writes
      const uint32_t from = two ? at_o : lanes + S::kTmemO;                   // (pipe 0's O, then pipe 1's)
      const float f0 = two || !pipe ? own : other, f1 = pipe ? own : other;
      if (busy) {
        char* out = p.out + (int64_t)(s.s0 + node) * p.out_n + head * p.out_h;
        float* part = scratch.sums(blockIdx.x, which) + (int64_t)row * HD;
#pragma unroll 1
        for (int d = d0; d < d1; d += 16) {
          uint32_t o[32];
          float y[16];
          tmem_load16x2(from + d, from + d + (single ? 0 : 128), o);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            y[i] = __uint_as_float(o[i]) * f0;
            if (!single) y[i] = fmaf(__uint_as_float(o[16 + i]), f1, y[i]);
          }
          if (r < rows) {
            if (aside) {
              float more[16];
              set_aside<DT, HD>(p, plans + seg % kPlans, aside, node, first, d, more);
#pragma unroll
              for (int i = 0; i < 16; ++i) y[i] += more[i];
            }
#pragma unroll
            for (int i = 0; i < 16; i += 8) {
              if (whole) {
                *reinterpret_cast<uint4*>(out + 2 * (d + i)) =
                    make_uint4(pack2<DT>(y[i], y[i + 1]), pack2<DT>(y[i + 2], y[i + 3]), pack2<DT>(y[i + 4], y[i + 5]), pack2<DT>(y[i + 6], y[i + 7]));
              } else {
                *reinterpret_cast<float4*>(part + d + i) = make_float4(y[i], y[i + 1], y[i + 2], y[i + 3]);
                *reinterpret_cast<float4*>(part + d + i + 4) = make_float4(y[i + 4], y[i + 5], y[i + 6], y[i + 7]);
              }
            }
          }
        }
      }
      if (r < rows && (two || pipe == 0)) {
        if (!whole) scratch.stats(blockIdx.x, which)[row] = make_float2(m, sum);
        else if (p.lse) p.lse[(int64_t)(s.s0 + node) * p.heads + head] = sum == 0.f ? -INFINITY : (m + log2f(sum)) * 0.6931471805599453f;
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(o_empty);
      if (!whole && s.x0 == 0) {
        wrote_start = true;
        if (tid == 0) *scratch.started(blockIdx.x) = Started{s.last, s.s0, s.row0, all, s.kvh};
      }
      read(seg);
      ++seg;  // (the next segment's maxima go where these ones are: enter() is a barrier)
    }
    asm volatile("cp.async.wait_all;" ::: "memory");  // (copies of Q are in flight only after a wait that ran out)
    if (!wrote_start && tid == 0) scratch.started(blockIdx.x)->last = 0;
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && *failed && p.status) atomicOr(p.status, AF_STATUS_TIMEOUT);
  if (*failed && (warp == kMmaS || warp == kMmaO)) {
    // After a wait has run out: the products that the two issue warps have in flight end before the CTA's tensor and shared
    // memory is given up (bounded): a commit follows the products of the thread that makes it.
    if (elect_one()) tc_commit(drained);
    __syncwarp();
    volatile int by_itself[2] = {0, kPatience};
    if (warp == kMmaS) wait_for(drained, 0, by_itself);
    __syncwarp();
  }
  if (warp == kMmaS) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int DT, int HD>
int launch(const Params& p, cudaStream_t s) {
  static_assert(Wide<HD>::kBytes <= 232448, "shared memory");
  if (int st = allow_smem<k_int4_attention_wide<DT, HD>>(Wide<HD>::kBytes, "af_tree_attention_int4")) return st;
  const int ctas = sm_count();
  cudaError_t e = launch_ex(k_int4_attention_wide<DT, HD>, dim3(ctas), dim3(kThreads), (size_t)Wide<HD>::kBytes, s, false, dim3(1), p);
  if (e == cudaSuccess && p.joins)
    e = launch_ex(k_join<DT, 2 * kRows, HD>, dim3(ctas, 32), dim3(kJoinThreads), 0, s, true, dim3(1), p, ctas);
  if (e != cudaSuccess) return fail(AF_ERR_CUDA, std::string("af_tree_attention_int4: launch: ") + cudaGetErrorString(e));
  return check_launch("af_tree_attention_int4");
}

}  // namespace

int wide_launch(const Params& p, bool bf16, int head_dim, cudaStream_t s) {
  if (head_dim == 128) return bf16 ? launch<AF_DTYPE_BF16, 128>(p, s) : launch<AF_DTYPE_F16, 128>(p, s);
  return bf16 ? launch<AF_DTYPE_BF16, 64>(p, s) : launch<AF_DTYPE_F16, 64>(p, s);
}

}  // namespace kv4
}  // namespace af
