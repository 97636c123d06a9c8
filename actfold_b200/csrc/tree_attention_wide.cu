// Attention of drafted trees with many rows per key/value head (sm_100a,
// tcgen05): the same work list, loads and joins as tree_attention.cu, but the
// rows are the M side (S [128 rows, 128 keys] = Q K^T, O += P V), because with
// more than 64 rows the tensor cores and the exponentials bound the work and
// not the keys that are read.
//
// A CTA holds two "pipes", each a 128-row O and a 128-row S of 128 keys, over
// which P is written in place (16 bits, TMEM operand of the second product).
// With more than 128 rows they are two row tiles over the same keys; with
// fewer, one row tile over the even and the odd key tiles, joined at the end.
// A thread owns a row, so no scores are exchanged: 64 of them at a time in
// registers, their maximum, the exponentials (128 x 128 of them take the SM's 16 per
// cycle 1024 cycles, as long as the two products of a tile), P back to TMEM. P V of
// the first 64 keys runs while the softmax works on the others (268 us without
// that, 255 us with S in halves too, whose products of 64 columns take as long as those
// of 128, 256 us so, for 4 requests of 64 nodes x 7 heads over up to 65 K keys). The
// reference maximum of a row is raised only when a score passes it by 2^8, as in
// the narrow kernel. Half of the exponentials as a polynomial on the multiply-add pipe made it
// slower (282 us).
//
// Measured on B200: that case 250 to 258 us in bursts (0.70 PFLOP/s), 291 to 296 us in long runs at
// the 1 kW power cap; ncu shows the tensor cores busy 40 %, the exponentials 40 %, DRAM
// 34 % (keys are read once per 256 rows): the chain of softmax, P V and Q K of two pipes bounds it.
//
// Warps 0-3 and 4-7: softmax of pipe 0 and 1; warp 8 loads Q and K, warp 9 V,
// warp 10 issues S, warp 11 plans and issues O.
#include "tree_attention.cuh"

namespace af {
namespace tree_attn {

namespace {

constexpr int kSoft = 8;
constexpr int kLoadK = kSoft, kLoadV = kSoft + 1, kMmaS = kSoft + 2, kMmaO = kSoft + 3;
constexpr int kThreads = (kSoft + 4) * 32;
constexpr int kRows = 128;  // of a row tile

template <int HD>
struct Wide {
  static constexpr int kHalves = HD / 64;
  static constexpr int kStage = kHalves * kHalf;                     // a K or V tile
  static constexpr int kKStages = 3, kVStages = 2;                   // V: see the wait for it below
  static constexpr int kOffK = 0, kOffV = kKStages * kStage;
  static constexpr int kQTiles = 2, kQRows = kRows, kQ = 1;
  static constexpr int kQBytes = kQTiles * kHalves * kRows * 128;
  static constexpr int kOffQ = kOffV + kVStages * kStage;
  static constexpr int kOffStat = kOffQ + kQBytes;                   // [2][128] (maximum, sum) of the pipes
  static constexpr int kOffBar = kOffStat + 2 * kRows * 8;
  static constexpr int kBars = 2 * kKStages + 2 * kVStages + 2 + 12 + 2 + kPlans + 1;
  static constexpr int kOffPlan = (kOffBar + kBars * 8 + 15) / 16 * 16;
  static constexpr int kBytes = kOffPlan + kPlans * 48 + 32;
  static constexpr int kTmemO = 2 * kKeys;                           // O of pipe x at kTmemO + 128 x, S of pipe x at 128 x
};

// 64 consecutive columns of the thread's TMEM lane.
__device__ __forceinline__ void tmem_load64(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%64];\n\ttcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]), "=r"(r[32]),
        "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]),
        "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]),
        "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]), "=r"(r[56]),
        "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
      : "r"(taddr)
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

// D [tmem] (+)= A [smem] * B [smem]^T (without the lane masks of tc_mma_bf16: a shorter issue).
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

template <int DT, int HD>
__global__ void __launch_bounds__(kThreads, 1) k_tree_attention_wide(const __grid_constant__ Params p) {
  using S = Wide<HD>;
  extern __shared__ __align__(1024) uint8_t gb[];
  pdl_trigger();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t base = smem_u32(gb);
  const uint32_t k_full = base + S::kOffBar, k_empty = k_full + 8 * S::kKStages, v_full = k_empty + 8 * S::kKStages,
                 v_empty = v_full + 8 * S::kVStages, q_full = v_empty + 8 * S::kVStages, q_empty = q_full + 8, s_full = q_empty + 8,
                 p_full = s_full + 32, done = p_full + 32, o_full = done + 32, o_empty = o_full + 8, plan_full = o_empty + 8,
                 drained = plan_full + 8 * kPlans;
  Segment* plans = reinterpret_cast<Segment*>(gb + S::kOffPlan);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(gb + S::kOffPlan + kPlans * 48);
  volatile int* failed = reinterpret_cast<volatile int*>(tmem_slot + 1);
  uint32_t* found = tmem_slot + 4;  // of even and of odd segments: tiles with values that are not finite

  if (tid == 0) {
    for (int i = 0; i < S::kKStages; ++i) {
      mbar_init(k_full + 8 * i, 1);
      mbar_init(k_empty + 8 * i, 1);
    }
    for (int i = 0; i < S::kVStages; ++i) {
      mbar_init(v_full + 8 * i, 1);
      mbar_init(v_empty + 8 * i, 1);
    }
    for (int i = 0; i < 4; ++i) {  // [pipe][half]
      mbar_init(s_full + 8 * i, 1);
      mbar_init(p_full + 8 * i, 4);
      mbar_init(done + 8 * i, 1);
    }
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    mbar_init(o_full, 1);
    mbar_init(o_empty, kSoft);
    for (int i = 0; i < kPlans; ++i) mbar_init(plan_full + 8 * i, 1);
    mbar_init(drained, 2);
    failed[0] = 0;
    failed[1] = p.patience;
    found[0] = found[1] = 0;
    fence_barrier_init();
  }
  if (warp == kMmaS) tmem_alloc(smem_u32(tmem_slot), 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const Scratch<2 * kRows, HD> scratch{p.ws, (int)gridDim.x};
  Segment s;
  auto planned = [&](int seg, Segment& s) { return read_plan(plans, plan_full, seg, s, failed); };
  auto agreed = [](bool mine) { return (bool)__all_sync(0xffffffffu, mine); };
  constexpr uint32_t kind = DT == AF_DTYPE_BF16 ? 0u : ((1u << 7) | (1u << 10));  // operand formats: bf16 = 1, f16 = 0

  if (warp == kLoadK) {
    load_tiles<S, false>(p, planned, base, k_full, k_empty, q_full, q_empty, failed);
  } else if (warp == kLoadV) {
    load_tiles<S, true>(p, planned, base, v_full, v_empty, q_full, q_empty, failed);
  } else if (warp == kMmaS) {
    // ---------------- S: two row tiles of a key tile, or one of every other key tile ----------------
    constexpr uint32_t id_s = idesc_bf16(kRows, kKeys) ^ kind;
    const uint64_t d_k = sw128_desc(base + S::kOffK), d_q = sw128_desc(base + S::kOffQ);
    bool ok = true;
    int seg = 0, stage = 0, k_phase = 0, used0 = 0, used1 = 0;  // tiles of S of the pipes
#pragma unroll 1
    while (ok && planned(seg, s)) {
      const bool two = s.n - s.node0 > p.nt_q;
      const int tiles = s.k1 - s.k0, steps = two ? 2 : 1;  // of a key tile
      ok = agreed(wait_for(q_full, seg & 1, failed));
#pragma unroll 1
      for (int t = 0; ok && t < tiles; ++t) {
        ok = agreed(wait_for(k_full + 8 * stage, k_phase, failed));
#pragma unroll 1
        for (int x = 0; ok && x < steps; ++x) {
          const int pipe = two ? x : t & 1, used = pipe ? used1 : used0;
          if (used) ok = agreed(wait_for(done + 8 * (2 * pipe + 1), (used - 1) & 1, failed));  // P V of the pipe's last keys
          if (!ok) break;
          tc_fence_after();
          const uint64_t a = d_q + (two && pipe ? (uint32_t)(S::kHalves * kRows * 128) >> 4 : 0u), b = d_k + (uint32_t)stage * (S::kStage >> 4);
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < HD / 16; ++kk)
              mma_from_smem(tmem + 128 * pipe, a + (kk >> 2) * (kRows * 8) + 2 * (kk & 3), b + (kk >> 2) * (kHalf >> 4) + 2 * (kk & 3), id_s,
                            kk ? 1u : 0u);
            tc_commit(s_full + 8 * pipe);
            if (x == steps - 1) tc_commit(k_empty + 8 * stage);
            if (x == steps - 1 && t == tiles - 1) tc_commit(q_empty);
          }
          __syncwarp();
        }
        used0 += two || !(t & 1);
        used1 += two || (t & 1);
        if (++stage == S::kKStages) {
          stage = 0;
          k_phase ^= 1;
        }
      }
      ++seg;
    }
    if (!ok) {
      *failed = 1;
      if (lane == 0 && p.status) atomicOr(p.status, AF_STATUS_TIMEOUT);
    }
  } else if (warp == kMmaO) {
    // ---------------- the plan, and O += P V of every half ----------------
    constexpr uint32_t id_o = idesc_bf16_bmn(kRows, HD) ^ kind;
    const uint64_t d_v = sw128_desc_mn(base + S::kOffV, kHalf, 1024);
    Planner planner;
    planner.begin(p, lane);
    planner.on(p, plans, plan_full, 1, lane);
    bool ok = true;
    int seg = 0, stage = 0, v_phase = 0, used0 = 0, used1 = 0;
#pragma unroll 1
    while (ok && planned(seg, s)) {
      // The plan that this one replaces has been read by everyone: the segment after it is done.
      planner.on(p, plans, plan_full, seg + 2, lane);
      const bool two = s.n - s.node0 > p.nt_q;
      const int tiles = s.k1 - s.k0, steps = two ? 4 : 2;
      if (seg > 0) ok = agreed(wait_for(o_empty, (seg - 1) & 1, failed));  // the last segment's O is read
#pragma unroll 1
      for (int t = 0; ok && t < tiles; ++t) {
        ok = agreed(wait_for(v_full + 8 * stage, v_phase, failed));
        const int keys16 = (s.pad + s.n - (s.k0 + t) * kKeys + 15) / 16;  // up to the row's last key
#pragma unroll 1
        for (int x = 0; ok && x < steps; ++x) {
          const int half = two ? x >> 1 : x, pipe = two ? x & 1 : t & 1, bar = 2 * pipe + half, used = pipe ? used1 : used0;
          ok = agreed(wait_for(p_full + 8 * bar, used & 1, failed));
          if (!ok) break;
          tc_fence_after();
          const uint64_t b = d_v + (uint32_t)stage * (S::kStage >> 4) + half * 4 * 128;
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
        if (++stage == S::kVStages) {
          stage = 0;
          v_phase ^= 1;
        }
      }
      ++seg;
    }
    if (!ok) {
      *failed = 1;
      if (lane == 0 && p.status) atomicOr(p.status, AF_STATUS_TIMEOUT);
    }
  } else {
    // ---------------- softmax of row r of the pipe's tiles ----------------
    const int quad = warp & 3, pipe = warp >> 2, r = 32 * quad + lane;
    const uint32_t lanes = tmem + ((uint32_t)(32 * quad) << 16);
    const uint32_t at_s = lanes + 128 * pipe, at_o = lanes + S::kTmemO + 128 * pipe;
    float2* stat = reinterpret_cast<float2*>(gb + S::kOffStat);
    const float sc = p.scale == 0.f ? 1.f : fabsf(p.scale);
    auto wait = [&](uint32_t bar, uint32_t parity) {
      if (!wait_for(bar, parity, failed)) *failed = 1;
    };
    int j0 = 0, seg = 0, taken = 0;  // tiles before this segment; halves of S of this pipe so far
    bool wrote_start = false;
    // Into the next segment go all softmax warps or none (see the narrow kernel).
    auto enter = [&]() {
      const bool there = planned(seg, s);
      return !vote_any<kSoft * 32>(1, !there || *failed);
    };
#pragma unroll 1
    while (enter()) {
      const bool two = s.n - s.node0 > p.nt_q;
      const int tiles = s.k1 - s.k0;
      const int first_node = s.node0 + (two && pipe ? p.nt_q : 0), rows = min(p.nt_q, s.n - first_node) * p.group;
      const int node = first_node + r / p.group;
      const bool busy = 32 * quad < rows;  // any of the warp's rows is one
      float m = kUnset;
      uint64_t l0 = 0ull, l1 = 0ull;
      uint32_t sick = 0;
#pragma unroll 1
      for (int x2 = two ? 0 : 2 * pipe; x2 < 2 * tiles; x2 += two || !(x2 & 1) ? 1 : 3, ++taken) {
        const int t = x2 >> 1, half = x2 & 1, bar = 2 * pipe + half;  // a half of a tile at a time
        const int key0 = (s.k0 + t) * kKeys;
        const bool masked = key0 + kKeys > s.len;
        if (half == 0) wait(s_full + 8 * pipe, (taken >> 1) & 1);
        tc_fence_after();
        if (masked && half == 0) {
          // Rows of V without a key, and drafted values that are not finite, are cleared (see the narrow kernel). S of
          // this tile follows products with the last V of this stage, so this wait is at most one phase ahead. With
          // two row tiles both pipes do it: each one's own writes are complete before its own P is.
          const int vt = j0 + t, key = key0 + r, x = key - s.pad;
          const bool in_prefix = key < s.len, in_tree = x >= 0 && x < s.n;
          wait(v_full + 8 * (vt % S::kVStages), (vt / S::kVStages) & 1);
          const uint32_t v_row = base + S::kOffV + vt % S::kVStages * S::kStage + r * 128;
          auto piece = [&](int c16) { return v_row + (c16 >> 3) * kHalf + 16 * ((c16 & 7) ^ (r & 7)); };
          if (!in_prefix && !in_tree && x < ((s.n + 15) & ~15) + 16) {
#pragma unroll 4
            for (int c16 = 0; c16 < 8 * S::kHalves; ++c16)
              asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(piece(c16)), "r"(0) : "memory");
          } else if (in_tree) {
            constexpr uint32_t e = DT == AF_DTYPE_BF16 ? 0x7f80u : 0x7c00u;
#pragma unroll 4
            for (int c16 = 0; c16 < 8 * S::kHalves; ++c16) {
              uint32_t w[4];
              asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(piece(c16)) : "memory");
              bool bad = false;
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const bool lo = (w[i] & e) == e, hi = ((w[i] >> 16) & e) == e;
                w[i] &= (lo ? 0u : 0xffffu) | (hi ? 0u : 0xffff0000u);
                bad |= lo || hi;
              }
              if (bad) {
                sick |= 1u << (t >> found_shift(tiles));
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(piece(c16)), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
              }
            }
          }
          fence_proxy_async_smem();
        }
        if (busy) {
          constexpr int C = kKeys / 2;
          uint32_t x[C];
          tmem_load64(at_s + C * half, x);
          if (p.scale <= 0.f) {  // scores in the order of the softmax
#pragma unroll
            for (int i = 0; i < C; ++i) x[i] = __float_as_uint(p.scale < 0.f ? -__uint_as_float(x[i]) : __uint_as_float(x[i]) * 0.f);
          }
          if (masked) {
#pragma unroll
            for (int c = 0; c < C / 32; ++c) {
              const int k = key0 + C * half + 32 * c, j = k - s.pad;  // the word's first key; as a node
              auto below = [](int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; };
              const uint32_t tree = below(s.n - j) & ~below(-j);
              const uint32_t vis = below(s.len - k) | (tree && r < rows ? seen_bits(p, s.s0, node, j) & tree : 0u);
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (!((vis >> i) & 1u)) x[32 * c + i] = 0xff800000u;
            }
          }
          float top[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            top[c] = __uint_as_float(x[16 * c]);
#pragma unroll
            for (int i = 1; i < 15; i += 2) top[c] = fmaxf(top[c], fmaxf(__uint_as_float(x[16 * c + i]), __uint_as_float(x[16 * c + i + 1])));
            top[c] = fmaxf(top[c], __uint_as_float(x[16 * c + 15]));
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
                tmem_load<8>(at_o + c, o);
#pragma unroll
                for (int i = 0; i < 8; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(at_o + c), "r"(o[0]), "r"(o[1]), "r"(o[2]),
                             "r"(o[3]), "r"(o[4]), "r"(o[5]), "r"(o[6]), "r"(o[7])
                             : "memory");
              }
            }
          }
          const uint64_t sc2 = pair(sc, sc), nm2 = pair(-m, -m);
          uint32_t e[C / 2];
#pragma unroll
          for (int i = 0; i < C / 2; i += 2) {
            const float2 a = unpair(fma2(pair(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1])), sc2, nm2));
            const float2 b = unpair(fma2(pair(__uint_as_float(x[2 * i + 2]), __uint_as_float(x[2 * i + 3])), sc2, nm2));
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
      // ---- the segment's rows ----
      const float2 la = unpair(add2(l0, l1));
      const float mine = la.x + la.y;
      stat[pipe * kRows + r] = make_float2(m, mine);
      if (sick) atomicOr(found + (seg & 1), sick);
      const bool set_aside = vote_any<kSoft * 32>(1, sick != 0);  // (and both pipes' maxima and sums are there)
      if (tid == 0) found[(seg + 1) & 1] = 0;  // (read last before this segment was entered)
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
      const int which = s.k0 == 0 ? 1 : 0;
      const float inv = !whole ? 1.f : sum == 0.f ? 0.f : 1.f / sum;
      own *= inv;
      other *= inv;
      const bool single = two || tiles == 1;  // only one pipe's O holds anything of these rows
      const int packed = (two && pipe ? p.nt_q * p.group : 0) + r;
      const int head = s.kvh * p.group + r % p.group;
      wait(o_full, seg & 1);
      tc_fence_after();
      const int d0 = two ? 0 : pipe * (HD / 2), d1 = two ? HD : d0 + HD / 2;  // the columns that this thread writes
      const uint32_t from = two ? at_o : lanes + S::kTmemO;                   // (pipe 0's O, then pipe 1's)
      const float f0 = two || !pipe ? own : other, f1 = pipe ? own : other;
      if (busy) {
        char* out = p.out + (int64_t)(s.s0 + node) * p.out_n + head * p.out_h;
        float* part = scratch.sums(blockIdx.x, which) + (int64_t)packed * HD;
#pragma unroll 1
        for (int d = d0; d < d1; d += 8) {
          uint32_t o[8];
          float y[8];
          tmem_load<8>(from + d, o);
#pragma unroll
          for (int i = 0; i < 8; ++i) y[i] = __uint_as_float(o[i]) * f0;
          if (!single) {
            tmem_load<8>(from + 128 + d, o);
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = fmaf(__uint_as_float(o[i]), f1, y[i]);
          }
          if (r < rows) {
            if (set_aside) {
              float more[8];
              set_aside_dims<DT>(p, plans + seg % kPlans, found + (seg & 1), node, d, more);
#pragma unroll
              for (int i = 0; i < 8; ++i) y[i] += more[i];
            }
            if (whole) {
              *reinterpret_cast<uint4*>(out + 2 * d) = make_uint4(pack2<DT>(y[0], y[1]), pack2<DT>(y[2], y[3]), pack2<DT>(y[4], y[5]), pack2<DT>(y[6], y[7]));
            } else {
              *reinterpret_cast<float4*>(part + d) = make_float4(y[0], y[1], y[2], y[3]);
              *reinterpret_cast<float4*>(part + d + 4) = make_float4(y[4], y[5], y[6], y[7]);
            }
          }
        }
      }
      if (r < rows && (two || pipe == 0)) {
        if (!whole) scratch.stats(blockIdx.x, which)[packed] = make_float2(m, sum);
        else if (p.lse) p.lse[(int64_t)(s.s0 + node) * p.heads + head] = sum == 0.f ? -INFINITY : (m + log2f(sum)) * 0.6931471805599453f;
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(o_empty);
      if (!whole && s.k0 == 0) {
        wrote_start = true;
        if (tid == 0) *scratch.started(blockIdx.x) = Started{s.last, s.s0 + s.node0, min(p.nt, s.n - s.node0) * p.group, s.kvh};
      }
      j0 += tiles;
      ++seg;  // (the next segment's maxima go where these ones are: enter() is a barrier)
    }
    if (!wrote_start && tid == 0) scratch.started(blockIdx.x)->last = 0;
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && *failed && p.status) atomicOr(p.status, AF_STATUS_TIMEOUT);
  if (*failed && (warp == kMmaS || warp == kMmaO)) drain_products(drained, warp == kMmaS);
  if (warp == kMmaS) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int DT, int HD>
int launch(const Params& p, cudaStream_t s) {
  static_assert(Wide<HD>::kBytes <= 232448, "shared memory");
  if (int st = allow_smem<k_tree_attention_wide<DT, HD>>(Wide<HD>::kBytes)) return st;
  const int ctas = sm_count();
  const cudaError_t e = launch_ex(k_tree_attention_wide<DT, HD>, dim3(ctas), dim3(kThreads), (size_t)Wide<HD>::kBytes, s, false, dim3(1), p);
  if (e != cudaSuccess) return fail(AF_ERR_CUDA, std::string("af_tree_attention: launch: ") + cudaGetErrorString(e));
  return join_launch<DT, 2 * kRows, HD>(p, ctas, s);
}

}  // namespace

int wide_launch(const Params& p, bool bf16, int head_dim, cudaStream_t s) {
  if (head_dim == 128) return bf16 ? launch<AF_DTYPE_BF16, 128>(p, s) : launch<AF_DTYPE_F16, 128>(p, s);
  return bf16 ? launch<AF_DTYPE_BF16, 64>(p, s) : launch<AF_DTYPE_F16, 64>(p, s);
}

}  // namespace tree_attn
}  // namespace af
