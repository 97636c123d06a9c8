// Attention of drafted trees over a paged key/value cache (sm_100a, tcgen05).
//
// For every request and key/value head, the rows (node, query head of the
// group) of its tree attend to the cached prefix and to the visible nodes of
// the tree. With few rows per head the work is one pass over the prefix's
// keys and values, so the products are transposed: the 128 KEYS of a tile are
// the M side of the tensor-core instruction and the rows (16 to 64 of them)
// its N side,
//   S^T [128 keys, rows] = K Q^T,       O^T [dim, rows] += V^T P^T,
// so a tile with 7 rows costs the exponentials of 8 rows, not of 128.
//
// Key positions of a request: its prefix [0, len), then its tree from
// pad = len rounded up to R, the rows of one TMA box (R <= 32 divides the page
// size), so a short tree shares the last tile of the prefix. All tiles of all
// (request, head, row tile) rows form one list, which the CTAs (one per SM)
// share evenly whatever the lengths are; a row that several CTAs worked on is
// joined by k_tree_attention_join from their partial sums.
//
// Warps 0-15 run the softmax: four groups of 128 threads (thread = key = TMEM
// lane), of which 1, 2 or 4 share the columns of a tile; the others work on the
// next tiles with maxima, sums and an O of their own (kPipes of them, joined at the
// end of a row), which hides the latency of a tile's chain of load, product,
// exponential, product. Warp 16 loads Q and K, warp 17 V (TMA; an issue takes
// some 60 cycles), warp 18 issues S, warp 19 plans the CTA's work and issues O. A column's
// reference maximum m is raised only when a score passes it by more than 2^8
// (or at the row's first key): steady tiles take one comparison per score and one
// barrier vote, no maximum across lanes. P then stays below 2^8 (2^15 in fp16, see
// kLead), rounded to 16 bits for the tensor cores: half a step of the type per
// probability. Sums and O are fp32. Every wait is
// bounded; a timeout sets AF_STATUS_TIMEOUT and all warps leave: the ones that meet at
// barriers by a common vote before each row (0.2 us of a call).
//
// Measured on B200 (128 dims, joins included): 64 requests of one token over 90 to
// 8000 keys, 28 heads over 4: 92.2 us, 5.8 TB/s of the 6.55 that a copy reaches. 8 trees of 20 to
// 64 nodes over 300 to 4100 keys, 32 heads: 78.8 us (4.2 TB/s; at every row's end the softmax warps,
// which write the output too, spend some 9000 cycles that no next row overlaps). One token over 523 keys:
// 12.6 us, all of it latency (plan, page table, first tile, five tiles, output) on 4 of the SMs.
#include "tree_attention.cuh"

namespace af {
namespace tree_attn {

namespace {

constexpr int kSoft = 16;                   // softmax warps
constexpr int kLoadK = kSoft, kLoadV = kSoft + 1, kMmaS = kSoft + 2, kMmaO = kSoft + 3;
constexpr int kThreads = (kSoft + 4) * 32;

// Shared memory: stages of (K, V) tiles, Q, and a little state. P^T of a tile
// goes over its keys, which nobody needs once S is there.
template <int N, int HD>
struct Shape {
  static constexpr int kCols = N < 32 ? N : 32;     // columns of a softmax thread
  static constexpr int kGroups = N / kCols;         // groups of 128 threads per tile
  static constexpr int kPipes = 4 / kGroups;        // tiles that are worked on at once
  static constexpr int kS = 4;                      // S buffers in TMEM
  static constexpr int kTmem = (kS + 2 * kPipes) * N <= 256 ? 256 : 512;  // S, then O [2 segments][kPipes]
  static constexpr int kHalves = HD / 64;
  static constexpr int kPitch = 2 * N;                        // bytes of a key's row of P^T
  static constexpr int kKBytes = kHalves * kHalf;             // (P^T, at most kHalf, goes over them)
  static constexpr int kStage = kKBytes + kHalves * kHalf;
  // At most kS, so that P of a tile is taken before P of the tile that uses the same barrier can be there: no wait is ever
  // two phases behind its barrier.
  static constexpr int kStages = (192 * 1024) / kStage < kS ? (192 * 1024) / kStage : kS;
  static constexpr int kQBytes = kHalves * N * 128;
  static constexpr int kQ = 2;                                // Q buffers
  // V lies before K: the second product always takes 128 dims, so with 64 it reads the 16 KB behind V too (for lanes of O
  // that nobody looks at), and those have to be there.
  static constexpr int kOffV = 0, kOffK = kHalves * kHalf, kKStages = kStages, kVStages = kStages, kQTiles = 1, kQRows = N;
  static_assert(N <= 64 && kOffK + kKBytes == kStage && kKBytes >= kHalf, "what the second product reads lies in its stage");
  static constexpr int kOffQ = kStages * kStage;
  static constexpr int kOffM = kOffQ + kQ * kQBytes;          // [kPipes][N] reference maxima, negated; then the factors of O
  static constexpr int kOffRed = kOffM + kPipes * N * 4;      // [kPipes][4][N] per-warp maxima or sums
  static constexpr int kOffBar = kOffRed + kPipes * 4 * N * 4;
  static constexpr int kBars = 3 * kStages + 4 + 3 * kS + 4 + kPlans + 1;
  static constexpr int kOffPlan = (kOffBar + kBars * 8 + 15) / 16 * 16;
  static constexpr int kBytes = kOffPlan + kPlans * 48 + 32;
};

// P^T [128 keys][N rows] in shared memory: rows of kPitch bytes whose 16-byte
// pieces are swizzled over as many bytes (32, 64 or 128).
template <int N>
__device__ __forceinline__ uint64_t p_desc(uint32_t at) {
  constexpr uint64_t pitch = 2 * N, swizzle = N == 16 ? 6 : N == 32 ? 4 : 2;
  return (uint64_t)((at & 0x3ffffu) >> 4) | (uint64_t)(kHalf >> 4) << 16 | (8 * pitch >> 4) << 32 | (uint64_t)1 << 46 | swizzle << 61;
}
template <int N>
__device__ __forceinline__ uint32_t p_piece(int key, int col) {  // byte offset of columns col .. col + 7 (a multiple of 8)
  constexpr int pieces = N / 8, shift = N == 16 ? 2 : N == 32 ? 1 : 0;
  return key * (16 * pieces) + 16 * ((col / 8) ^ ((key >> shift) % pieces));
}

// Lane i's 32 bits become bit i of every lane's word.
__device__ __forceinline__ uint32_t transpose_bits(uint32_t x, int lane) {
#pragma unroll
  for (uint32_t k = 16, m = 0x0000ffffu; k > 0; k >>= 1, m ^= m << k) {
    const uint32_t y = __shfl_xor_sync(0xffffffffu, x, k);
    x = lane & k ? ((y >> k) & m) | (x & ~m) : (x & m) | ((y & m) << k);
  }
  return x;
}

// W columns (4 or 8) of each of P blocks of N columns.
template <int P, int N, int W>
__device__ __forceinline__ void tmem_load_rows(uint32_t taddr, uint32_t* r) {
#define AF_LD4(a, b) "tcgen05.ld.sync.aligned.32x32b.x4.b32 {" a "}, [" b "];\n\t"
#define AF_LD8(a, b) "tcgen05.ld.sync.aligned.32x32b.x8.b32 {" a "}, [" b "];\n\t"
  static_assert((P == 2 && W == 8) || P == 4, "pipes");
  if constexpr (P == 2) {
    asm volatile(AF_LD8("%0,%1,%2,%3,%4,%5,%6,%7", "%16") AF_LD8("%8,%9,%10,%11,%12,%13,%14,%15", "%17") "tcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                   "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr), "r"(taddr + N)
                 : "memory");
  } else if constexpr (W == 4) {
    asm volatile(AF_LD4("%0,%1,%2,%3", "%16") AF_LD4("%4,%5,%6,%7", "%17") AF_LD4("%8,%9,%10,%11", "%18")
                     AF_LD4("%12,%13,%14,%15", "%19") "tcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                   "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr), "r"(taddr + N), "r"(taddr + 2 * N), "r"(taddr + 3 * N)
                 : "memory");
  } else {
    asm volatile(AF_LD8("%0,%1,%2,%3,%4,%5,%6,%7", "%32") AF_LD8("%8,%9,%10,%11,%12,%13,%14,%15", "%33")
                     AF_LD8("%16,%17,%18,%19,%20,%21,%22,%23", "%34") AF_LD8("%24,%25,%26,%27,%28,%29,%30,%31", "%35")
                         "tcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                   "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
                   "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
                   "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(taddr), "r"(taddr + N), "r"(taddr + 2 * N), "r"(taddr + 3 * N)
                 : "memory");
  }
#undef AF_LD4
#undef AF_LD8
}
__device__ __forceinline__ void tmem_store8(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

// C values per lane (16 or 32) reduced across the warp: lane x returns the
// result of value x * C / 32. Each step halves the values that a lane keeps
// (C - 1 exchanges and one more where C is 16; a reduction per value takes 5 C).
template <int C, typename Op>
__device__ __forceinline__ float transpose_reduce(float* v, int lane, Op op) {
#pragma unroll
  for (int o = 16, n = C / 2; n > 0; o >>= 1, n >>= 1) {
    const bool up = (lane & o) != 0;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const float give = up ? v[i] : v[i + n], keep = up ? v[i + n] : v[i];
      v[i] = op(keep, __shfl_xor_sync(0xffffffffu, give, o));
    }
  }
  return C == 32 ? v[0] : op(v[0], __shfl_xor_sync(0xffffffffu, v[0], 1));
}

template <int DT, int N, int HD>
__global__ void __launch_bounds__(kThreads, 1) k_tree_attention(const __grid_constant__ Params p) {
  using S = Shape<N, HD>;
  extern __shared__ __align__(1024) uint8_t gb[];
  pdl_trigger();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t base = smem_u32(gb), sQ = base + S::kOffQ;
  const uint32_t k_full = base + S::kOffBar, v_full = k_full + 8 * S::kStages, empty = v_full + 8 * S::kStages, q_full = empty + 8 * S::kStages,
                 q_empty = q_full + 16, s_full = q_empty + 16, p_full = s_full + 8 * S::kS, done = p_full + 8 * S::kS, o_full = done + 8 * S::kS,
                 o_empty = o_full + 16, plan_full = o_empty + 16, drained = plan_full + 8 * kPlans;
  Segment* plans = reinterpret_cast<Segment*>(gb + S::kOffPlan);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(gb + S::kOffPlan + kPlans * 48);
  volatile int* failed = reinterpret_cast<volatile int*>(tmem_slot + 1);
  uint32_t* found = tmem_slot + 4;  // of even and of odd segments: tiles with values that are not finite
  static_assert(sizeof(Segment) == 48, "plans");

  if (tid == 0) {
    for (int i = 0; i < S::kStages; ++i) {
      mbar_init(k_full + 8 * i, 1);
      mbar_init(v_full + 8 * i, 1);
      mbar_init(empty + 8 * i, 1);
    }
    for (int i = 0; i < S::kS; ++i) {
      mbar_init(s_full + 8 * i, 1);
      mbar_init(p_full + 8 * i, 4 * S::kGroups);
      mbar_init(done + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(q_full + 8 * i, 1);
      mbar_init(q_empty + 8 * i, 1);
      mbar_init(o_full + 8 * i, 1);
      mbar_init(o_empty + 8 * i, kSoft);
    }
    for (int i = 0; i < kPlans; ++i) mbar_init(plan_full + 8 * i, 1);
    mbar_init(drained, 2);
    failed[0] = 0;
    failed[1] = p.patience;
    found[0] = found[1] = 0;
    fence_barrier_init();
  }
  if (warp == kMmaS) tmem_alloc(smem_u32(tmem_slot), S::kTmem);

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const Scratch<N, HD> scratch{p.ws, (int)gridDim.x};
  Segment s;
  auto planned = [&](int seg, Segment& s) { return read_plan(plans, plan_full, seg, s, failed); };
  constexpr uint32_t kind = DT == AF_DTYPE_BF16 ? 0u : ((1u << 7) | (1u << 10));  // operand formats: bf16 = 1, f16 = 0
  auto agreed = [](bool mine) { return (bool)__all_sync(0xffffffffu, mine); };

  if (warp == kLoadK) {
    load_tiles<S, false>(p, planned, base, k_full, empty, q_full, q_empty, failed);
  } else if (warp == kLoadV) {
    load_tiles<S, true>(p, planned, base, v_full, empty, q_full, q_empty, failed);
  } else if (warp == kMmaS) {
    // ---------------- S^T of every tile ----------------
    // The whole warp keeps the books, one lane issues: descriptors stay in uniform registers.
    constexpr uint32_t id_s = idesc_bf16(kKeys, N) ^ kind;
    const uint64_t d_k = sw128_desc(base + S::kOffK), d_q = sw128_desc(sQ);
    bool ok = true;
    int j = 0, seg = 0, stage = 0, stage_phase = 0;
#pragma unroll 1
    while (ok && planned(seg, s)) {
      const int qb = seg % S::kQ;
      ok = agreed(wait_for(q_full + 8 * qb, (seg / S::kQ) & 1, failed));
      const uint64_t b = d_q + (uint32_t)qb * (S::kQBytes >> 4);
#pragma unroll 1
      for (int kt = s.k0; ok && kt < s.k1; ++kt, ++j) {
        const int sb = j % S::kS;
        ok = agreed(wait_for(k_full + 8 * stage, stage_phase, failed));
        if (ok && j >= S::kS) ok = agreed(wait_for(p_full + 8 * sb, (j / S::kS - 1) & 1, failed));  // S buffer sb is read
        if (!ok) break;
        tc_fence_after();
        const uint64_t a = d_k + (uint32_t)stage * (S::kStage >> 4);
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk)
            tc_mma_bf16(tmem + sb * N, a + (kk >> 2) * (kHalf >> 4) + 2 * (kk & 3), b + (kk >> 2) * (N * 8) + 2 * (kk & 3), id_s, kk ? 1u : 0u);
          tc_commit(s_full + 8 * sb);
          if (kt + 1 == s.k1) tc_commit(q_empty + 8 * qb);
        }
        __syncwarp();
        if (++stage == S::kStages) {
          stage = 0;
          stage_phase ^= 1;
        }
      }
      ++seg;
    }
    if (!ok) {
      *failed = 1;
      if (lane == 0 && p.status) atomicOr(p.status, AF_STATUS_TIMEOUT);
    }
  } else if (warp == kMmaO) {
    // ---------------- O^T += V^T P^T of every tile, into its pipe's O ----------------
    constexpr uint32_t id_o = (idesc_bf16(128, N) ^ kind) | (1u << 15) | (1u << 16);  // A and B MN-major
    const uint64_t d_v = sw128_desc_mn(base + S::kOffV, kHalf, 1024), d_p = p_desc<N>(base + S::kOffK);
    bool ok = true;
    int j = 0, seg = 0, stage = 0, stage_phase = 0;
    Planner planner;
    planner.begin(p, lane);
    planner.on(p, plans, plan_full, 1, lane);
#pragma unroll 1
    while (ok && planned(seg, s)) {
      // Everyone is done with the plan that this one replaces: P of the segment before this one is there.
      planner.on(p, plans, plan_full, seg + 2, lane);
      const int ob = seg & 1;
      if (seg >= 2) ok = agreed(wait_for(o_empty + 8 * ob, ((seg >> 1) - 1) & 1, failed));
#pragma unroll 1
      for (int kt = s.k0; ok && kt < s.k1; ++kt, ++j) {
        const int sb = j % S::kS, pipe = j % S::kPipes;
        ok = agreed(wait_for(v_full + 8 * stage, stage_phase, failed)) && agreed(wait_for(p_full + 8 * sb, (j / S::kS) & 1, failed));
        if (!ok) break;
        tc_fence_after();
        const uint64_t a = d_v + (uint32_t)stage * (S::kStage >> 4), b = d_p + (uint32_t)stage * (S::kStage >> 4);
        const uint32_t o = tmem + (S::kS + ob * S::kPipes + pipe) * N;
        const uint32_t add = kt - s.k0 < S::kPipes ? 0u : 1u;
        const int steps = min(kKeys / 16, (s.pad + s.n - kt * kKeys + 15) / 16);  // up to the row's last key
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < kKeys / 16; ++kk)
            if (kk < steps) tc_mma_bf16(o, a + kk * 128, b + kk * S::kPitch, id_o, kk ? 1u : add);
          tc_commit(empty + 8 * stage);
          tc_commit(done + 8 * sb);
          if (kt + 1 == s.k1) tc_commit(o_full + 8 * ob);
        }
        __syncwarp();
        if (++stage == S::kStages) {
          stage = 0;
          stage_phase ^= 1;
        }
      }
      ++seg;
    }
    if (!ok) {
      *failed = 1;
      if (lane == 0 && p.status) atomicOr(p.status, AF_STATUS_TIMEOUT);
    }
  } else {
    // ---------------- softmax: key 32 * quad + lane, columns c0 .. c0 + C - 1 of its pipe's tiles ----------------
    constexpr int C = S::kCols, kTeam = 128;
    const int quad = warp & 3, wg = warp >> 2, pipe = wg / S::kGroups, r = 32 * quad + lane, c0 = wg % S::kGroups * C;
    const int team = 1 + wg, team_tid = tid - kTeam * wg;  // barrier of the threads with the same columns
    const uint32_t lanes = tmem + ((uint32_t)(32 * quad) << 16);
    float* m_all = reinterpret_cast<float*>(gb + S::kOffM);
    float* red_all = reinterpret_cast<float*>(gb + S::kOffRed);
    float* fac = m_all;
    float* m_neg = m_all + pipe * N + c0;        // -(reference maximum) of the thread's columns
    float* red = red_all + pipe * 4 * N + c0;    // red[quad * N + column]; row 0: factors of the old O
    const int red_at = quad * N + lane * C / 32;
    const uint64_t scale2 = pair(p.scale, p.scale);
    auto wait = [&](uint32_t bar, uint32_t parity) {
      if (!wait_for(bar, parity, failed)) *failed = 1;
    };
    int j0 = 0, seg = 0;  // tiles before this segment
    bool wrote_start = false;
    // Into the next segment go all softmax warps or none, whatever each has seen of a plan or of a wait that ran out: the
    // barriers inside have no limit of their own.
    auto enter = [&]() {
      const bool there = planned(seg, s);
      return !vote_any<kSoft * 32>(5, !there || *failed);
    };
#pragma unroll 1
    while (enter()) {
      const int cols = min(p.nt, s.n - s.node0) * p.group;
      const int live = min(C, max(0, cols - c0));  // columns of this thread that are rows
      uint64_t l[C / 2];                           // this key's part of the sums
#pragma unroll
      for (int i = 0; i < C / 2; ++i) l[i] = 0ull;
      if (team_tid < C) m_neg[team_tid] = -kUnset;
      uint32_t sick = 0;   // tiles whose drafted values that are not finite were set aside (see found_shift)
      bool begun = false;  // this pipe's O holds something
      named_bar_sync(team, kTeam);
      const int tiles = s.k1 - s.k0;
#pragma unroll 1
      for (int i0 = (pipe + S::kPipes - j0 % S::kPipes) % S::kPipes; i0 < tiles; i0 += S::kPipes) {
        const int j = j0 + i0, sb = j % S::kS, stage = j % S::kStages;
        const int key0 = (s.k0 + i0) * kKeys, key = key0 + r, node = key - s.pad;
        const bool masked = key0 + kKeys > s.len;
        const bool in_prefix = key < s.len, in_tree = node >= 0 && node < s.n;
        const uint32_t stage_at = base + stage * S::kStage;
        uint32_t vis = 0xffffffffu;  // bit i: column c0 + i sees this key
        if (masked) {  // (read while S is on its way)
          const int c = c0 + lane;
          vis = transpose_bits(lane < C && c < cols ? seen_bits(p, s.s0, s.node0 + c / p.group, node - lane) : 0u, lane);
          vis = in_prefix ? 0xffffffffu : in_tree ? vis : 0u;
        }
        // S of this tile also says that its stage was loaded, so the wait for its V below is at most one phase ahead.
        wait(s_full + 8 * sb, (j / S::kS) & 1);
        tc_fence_after();
        if (masked) {
          // Rows of V without a key (of those that the product takes) are whatever lay there: cleared. A drafted value that is not finite would reach
          // every column as 0 * inf: it is cleared too, and added at the end to the columns that see it.
          wait(v_full + 8 * stage, (j / S::kStages) & 1);
          const uint32_t v_row = stage_at + S::kOffV + r * 128;
          auto piece = [&](int c16) { return v_row + (c16 >> 3) * kHalf + 16 * ((c16 & 7) ^ (r & 7)); };
          if (!in_prefix && !in_tree && node < ((s.n + 15) & ~15) + 16) {
#pragma unroll 4
            for (int c16 = c0 / C; c16 < 8 * S::kHalves; c16 += S::kGroups)
              asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(piece(c16)), "r"(0) : "memory");
          } else if (in_tree && (s.n > 1 || p.mask)) {  // (the node of a chain of one is hidden from nobody)
            constexpr uint32_t e = DT == AF_DTYPE_BF16 ? 0x7f80u : 0x7c00u;
#pragma unroll 4
            for (int c16 = c0 / C; c16 < 8 * S::kHalves; c16 += S::kGroups) {
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
                sick |= 1u << (i0 >> found_shift(tiles));
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(piece(c16)), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
              }
            }
          }
        }
        uint32_t x[C];
        // x = score - reference maximum (in log2 units); hidden scores -inf.
        float top = -INFINITY;
        auto shift = [&]() {
          tmem_load<C>(lanes + sb * N + c0, x);
#pragma unroll
          for (int q8 = 0; q8 < C / 8; ++q8) {
            if (8 * q8 < live) {
#pragma unroll
              for (int q = 8 * q8; q < 8 * q8 + 8; q += 4) {
                const ulonglong2 m = *reinterpret_cast<const ulonglong2*>(m_neg + q);
                const float2 y0 = unpair(fma2(pair(__uint_as_float(x[q]), __uint_as_float(x[q + 1])), scale2, m.x));
                const float2 y1 = unpair(fma2(pair(__uint_as_float(x[q + 2]), __uint_as_float(x[q + 3])), scale2, m.y));
                x[q] = __float_as_uint(y0.x);
                x[q + 1] = __float_as_uint(y0.y);
                x[q + 2] = __float_as_uint(y1.x);
                x[q + 3] = __float_as_uint(y1.y);
                top = fmaxf(top, fmaxf(y0.x, y0.y));
                top = fmaxf(top, fmaxf(y1.x, y1.y));
              }
            }
          }
          if (masked) {
            top = -INFINITY;
#pragma unroll
            for (int i = 0; i < C; ++i) {
              if (!((vis >> i) & 1u)) x[i] = 0xff800000u;
              if (i < live) top = fmaxf(top, __uint_as_float(x[i]));
            }
          }
        };
        if (begun) shift();
        if (!begun || vote_any<kTeam>(team, top > kLead<DT> + kRaise)) {
          // New maxima of the columns that need one (at first of all of them), from the scores themselves.
          tmem_load<C>(lanes + sb * N + c0, x);
          float y[C];
#pragma unroll
          for (int i = 0; i < C; ++i) y[i] = (vis >> i) & 1u ? __uint_as_float(x[i]) * p.scale : -INFINITY;
          red[red_at] = transpose_reduce<C>(y, lane, [](float a, float b) { return fmaxf(a, b); });
          named_bar_sync(team, kTeam);
          if (team_tid < C) {
            const float t = fmaxf(fmaxf(red[team_tid], red[N + team_tid]), fmaxf(red[2 * N + team_tid], red[3 * N + team_tid]));
            const float old = -m_neg[team_tid];
            const bool raise = old == kUnset ? t > kUnset : t > old + (kLead<DT> + kRaise);
            red[team_tid] = raise ? (old == kUnset ? 0.f : exp2f(old - (t - kLead<DT>))) : 1.f;
            if (raise) m_neg[team_tid] = kLead<DT> - t;
          }
          named_bar_sync(team, kTeam);
          if (begun) {
            // O of the pipe's tiles before this one is complete once the last one's product is.
            const int jb = j - S::kPipes;
            wait(done + 8 * (jb % S::kS), (jb / S::kS) & 1);
            tc_fence_after();
#pragma unroll
            for (int q8 = 0; q8 < C / 8; ++q8) {
              if (8 * q8 < live) {
                uint32_t o[8];
                const uint32_t addr = lanes + (S::kS + (seg & 1) * S::kPipes + pipe) * N + c0 + 8 * q8;
                tmem_load<8>(addr, o);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const float2 f = *reinterpret_cast<const float2*>(red + 8 * q8 + 2 * i);
                  o[2 * i] = __float_as_uint(__uint_as_float(o[2 * i]) * f.x);
                  o[2 * i + 1] = __float_as_uint(__uint_as_float(o[2 * i + 1]) * f.y);
                  l[4 * q8 + i] = fma2(l[4 * q8 + i], pair(f.x, f.y), 0ull);
                }
                tmem_store8(addr, o);
              }
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
          }
          shift();
        }
        begun = true;
        // P^T row of this key: 16-byte pieces of 8 columns.
#pragma unroll
        for (int q8 = 0; q8 < C / 8; ++q8) {
          if (8 * q8 < live) {
            float e[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = ex2(__uint_as_float(x[8 * q8 + i]));
#pragma unroll
            for (int i = 0; i < 4; ++i) l[4 * q8 + i] = add2(l[4 * q8 + i], pair(e[2 * i], e[2 * i + 1]));
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage_at + S::kOffK + p_piece<N>(r, c0 + 8 * q8)), "r"(pack2<DT>(e[0], e[1])),
                         "r"(pack2<DT>(e[2], e[3])), "r"(pack2<DT>(e[4], e[5])), "r"(pack2<DT>(e[6], e[7]))
                         : "memory");
          }
        }
        fence_proxy_async_smem();  // P (and V) are read by the tensor cores
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full + 8 * sb);
      }
      // ---- the segment's rows: the pipes' sums and O joined; O^T lane = dim, column = row ----
      const bool whole = s.whole != 0;
      const int which = s.k0 == 0 ? 1 : 0;
      const int64_t first = s.s0 + (int64_t)s.node0;
      named_bar_sync(team, kTeam);  // the last factors are read
      {
        float y[C];
#pragma unroll
        for (int i = 0; i < C / 2; ++i) {
          const float2 v = unpair(l[i]);
          y[2 * i] = v.x;
          y[2 * i + 1] = v.y;
        }
        const float sum = transpose_reduce<C>(y, lane, [](float a, float b) { return a + b; });
        red[red_at] = sum;
      }
      if (sick) atomicOr(found + (seg & 1), sick);
      const bool set_aside = vote_any<kSoft * 32>(5, sick != 0);  // (and the sums are there)
      if (tid == 0) found[(seg + 1) & 1] = 0;  // (read last before this segment was entered)
      if (tid < cols) {
        float m = kUnset, sum = 0.f, f[S::kPipes];
#pragma unroll
        for (int q = 0; q < S::kPipes; ++q) m = fmaxf(m, -m_all[q * N + tid]);
#pragma unroll
        for (int q = 0; q < S::kPipes; ++q) {
          const float* lq = red_all + q * 4 * N + tid;
          f[q] = -m_all[q * N + tid] == m ? 1.f : exp2f(-m_all[q * N + tid] - m);
          sum += f[q] * ((lq[0] + lq[N]) + (lq[2 * N] + lq[3 * N]));
        }
        const float inv = !whole ? 1.f : sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
        for (int q = 0; q < S::kPipes; ++q) fac[q * N + tid] = f[q] * inv;
        if (!whole) scratch.stats(blockIdx.x, which)[tid] = make_float2(m, sum);
        else if (p.lse)
          p.lse[(first + tid / p.group) * p.heads + s.kvh * p.group + tid % p.group] =
              sum == 0.f ? -INFINITY : (m + log2f(sum)) * 0.6931471805599453f;
      }
      wait(o_full + 8 * (seg & 1), (seg >> 1) & 1);
      tc_fence_after();
      named_bar_sync(5, kSoft * 32);
      constexpr int kOut = N / 4, kW = kOut < 8 ? kOut : 8;  // columns that a group of 128 threads writes, and at once
      const int o0 = wg * kOut, o1 = min(cols, o0 + kOut);
      if (32 * quad < HD && o0 < o1) {
        float* part = scratch.sums(blockIdx.x, which) + r;
        int i = o0 / p.group, head = o0 - i * p.group;
        char* out = p.out + (first + i) * p.out_n + (s.kvh * p.group + head) * p.out_h + 2 * r;
        const int64_t wrap = p.out_n - (p.group - 1) * p.out_h;  // from a node's last head to the next node's first
        uint32_t there = 0;  // the pipes with a tile of this segment (the O of another one is anything)
#pragma unroll
        for (int q = 0; q < S::kPipes; ++q) there |= (uint32_t)((q + S::kPipes - j0 % S::kPipes) % S::kPipes < tiles) << q;
#pragma unroll 1
        for (int c8 = o0; c8 < o1; c8 += kW) {
          float y[kW];
          uint32_t o[kW * S::kPipes];
          tmem_load_rows<S::kPipes, N, kW>(lanes + (S::kS + (seg & 1) * S::kPipes) * N + c8, o);
#pragma unroll
          for (int e = 0; e < kW; ++e) y[e] = 0.f;
#pragma unroll
          for (int q = 0; q < S::kPipes; ++q) {
            if ((there >> q) & 1u) {
#pragma unroll
              for (int e = 0; e < kW; e += 4) {
                const float4 f = *reinterpret_cast<const float4*>(fac + q * N + c8 + e);
                y[e] = fmaf(__uint_as_float(o[kW * q + e]), f.x, y[e]);
                y[e + 1] = fmaf(__uint_as_float(o[kW * q + e + 1]), f.y, y[e + 1]);
                y[e + 2] = fmaf(__uint_as_float(o[kW * q + e + 2]), f.z, y[e + 2]);
                y[e + 3] = fmaf(__uint_as_float(o[kW * q + e + 3]), f.w, y[e + 3]);
              }
            }
          }
          if (set_aside) {
            float more[kW];
            set_aside_rows<DT, kW>(p, plans + seg % kPlans, found + (seg & 1), c8, min(o1, c8 + kW), r, more);
#pragma unroll
            for (int e = 0; e < kW; ++e) y[e] += more[e];
          }
          if (whole) {
#pragma unroll
            for (int e = 0; e < kW; ++e) {
              if (c8 + e < o1) *reinterpret_cast<uint16_t*>(out) = to_bits<DT>(y[e]);
              const bool next = ++head == p.group;
              out += next ? wrap : p.out_h;
              head = next ? 0 : head;
            }
          } else {
#pragma unroll
            for (int e = 0; e < kW; ++e)
              if (c8 + e < o1) part[(c8 + e) * HD] = y[e];
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(o_empty + 8 * (seg & 1));
      if (!whole && s.k0 == 0) {
        wrote_start = true;
        if (tid == 0) *scratch.started(blockIdx.x) = Started{s.last, (int)first, cols, s.kvh};
      }
      j0 += tiles;
      ++seg;  // (the factors lie where the next maxima go: enter() is a barrier)
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
    tmem_dealloc(tmem, S::kTmem);
  }
}

constexpr int kJoinThreads = 256;
template <int N>
constexpr int kJoinBlocks = N <= 64 ? 8 : 16;  // per CTA of the main kernel (8: all of them resident at once)

// Rows that several CTAs worked on: out = sum_c w_c O_c / sum_c w_c l_c with
// w_c = 2^(m_c - max m), in the CTAs' order. The block's 8 warps share a row's
// parts where there are many, and take a row each where there are few.
template <int DT, int N, int HD>
__global__ void __launch_bounds__(kJoinThreads) k_tree_attention_join(const __grid_constant__ Params p, int ctas) {
  constexpr int V = HD / 32, W = kJoinThreads / 32;
  __shared__ float acc[W][HD + 1];
  pdl_wait();
  const Scratch<N, HD> scratch{p.ws, ctas};
  const int c = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Started st = *scratch.started(c);
  if (st.last <= c) return;
  const int parts = st.last - c + 1;
  const bool share = parts > 8;
  for (int row = share ? blockIdx.y : blockIdx.y * W + warp; row < st.rows; row += share ? kJoinBlocks<N> : kJoinBlocks<N> * W) {
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
      // A part without a key has weight 0 and sums of 0.
#pragma unroll
      for (int v = 0; v < V; ++v) y[v] += w * o[v];
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
      const int64_t node = st.node0 + row / p.group;
      const int head = st.kvh * p.group + row % p.group;
#pragma unroll
      for (int v = 0; v < V; ++v) y[v] = sum == 0.f ? 0.f : y[v] / sum;
      uint32_t* out = reinterpret_cast<uint32_t*>(p.out + node * p.out_n + head * p.out_h) + lane * (V / 2);
#pragma unroll
      for (int v = 0; v < V / 2; ++v) out[v] = pack2<DT>(y[2 * v], y[2 * v + 1]);
      if (lane == 0 && p.lse) p.lse[node * p.heads + head] = sum == 0.f ? -INFINITY : (m + log2f(sum)) * 0.6931471805599453f;
    }
  }
}

std::atomic<int> g_patience{kPatience};

int64_t workspace_bytes() { return Scratch<256, 128>::bytes(sm_count()); }

int check_args(const af_tree_attention_args& a) {
  AF_REQUIRE(a.batch >= 0 && a.total >= 0 && a.max_pages >= 0 && a.pages >= 0, "af_tree_attention: bad shape");
  AF_REQUIRE(a.n_heads > 0 && a.n_kv_heads > 0 && a.n_heads % a.n_kv_heads == 0, "af_tree_attention: n_heads must be a multiple of n_kv_heads");
  AF_REQUIRE(a.n_heads / a.n_kv_heads <= 64, "af_tree_attention: at most 64 query heads per key/value head");
  AF_REQUIRE(a.head_dim == 64 || a.head_dim == 128, "af_tree_attention: head_dim must be 64 or 128");
  AF_REQUIRE(a.dtype == AF_DTYPE_F16 || a.dtype == AF_DTYPE_BF16, "af_tree_attention: dtype must be fp16 or bf16");
  AF_REQUIRE(a.page_size > 0 && a.page_size % 8 == 0 && a.page_size <= (1 << 20), "af_tree_attention: page_size must be a multiple of 8");
  AF_REQUIRE(a.batch <= AF_TREE_ATTN_MAX_BATCH, "af_tree_attention: at most 16384 requests");
  AF_REQUIRE(a.total <= (1 << 28) && a.pages <= 0x7fffffff && a.n_heads <= (1 << 16) && a.max_pages <= (1 << 30) && a.max_pages * a.page_size <= (1 << 30),
             "af_tree_attention: size too large");
  AF_REQUIRE(!a.mask || (a.words > 0 && a.words <= AF_TREE_MAX_NODES / 32 && a.mask_stride >= a.words), "af_tree_attention: bad mask");
  if (a.batch == 0 || a.total == 0) return AF_OK;
  AF_REQUIRE(a.q && a.k && a.v && a.out && a.lengths && a.starts && a.workspace, "af_tree_attention: null pointer");
  AF_REQUIRE(a.max_pages == 0 || a.pages == 0 || (a.k_cache && a.v_cache && a.tables), "af_tree_attention: null pointer");
  uint64_t al = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v) |
                reinterpret_cast<uintptr_t>(a.k_cache) | reinterpret_cast<uintptr_t>(a.v_cache) | reinterpret_cast<uintptr_t>(a.out) |
                reinterpret_cast<uintptr_t>(a.workspace);
  for (int i = 0; i < 2; ++i)
    al |= (uint64_t)a.q_strides[i] | (uint64_t)a.k_strides[i] | (uint64_t)a.v_strides[i] | (uint64_t)a.out_strides[i];
  for (int i = 0; i < 3; ++i) al |= (uint64_t)a.k_cache_strides[i] | (uint64_t)a.v_cache_strides[i];
  const struct {
    int64_t n, stride;
  } dims[] = {{a.total, a.q_strides[0]},         {a.n_heads, a.q_strides[1]},         {a.total, a.k_strides[0]},
              {a.n_kv_heads, a.k_strides[1]},    {a.total, a.v_strides[0]},           {a.n_kv_heads, a.v_strides[1]},
              {a.pages, a.k_cache_strides[0]},   {a.page_size, a.k_cache_strides[1]}, {a.n_kv_heads, a.k_cache_strides[2]},
              {a.pages, a.v_cache_strides[0]},   {a.page_size, a.v_cache_strides[1]}, {a.n_kv_heads, a.v_cache_strides[2]},
              {a.total, a.out_strides[0]},       {a.n_heads, a.out_strides[1]}};
  for (const auto& d : dims)
    AF_REQUIRE(d.n <= 1 || (d.stride > 0 && d.stride < (1LL << 40)), "af_tree_attention: strides must be positive and below 2^40");
  AF_REQUIRE(a.workspace_bytes >= workspace_bytes(), "af_tree_attention: the workspace is too small");
  AF_REQUIRE((al & 15) == 0, "af_tree_attention: addresses and strides must be multiples of 16 bytes");
  return AF_OK;
}

// A map of `rank` dimensions (innermost first; strides of the others in
// bytes), boxes of 64 x the given extents, 128-byte swizzle, zeros outside.
int tree_map(CUtensorMap* map, const void* base, int dtype, int rank, const uint64_t* dims, const int64_t* strides, const uint32_t* box) {
  uint64_t st[4];
  for (int i = 0; i + 1 < rank; ++i) st[i] = strides[i] ? (uint64_t)strides[i] : dims[0] * 2;  // of a single entry: any
  return make_tmap_strided16(map, base, dtype == AF_DTYPE_BF16, rank, dims, st, box);
}

template <int DT, int N, int HD>
int launch(const Params& p, cudaStream_t s) {
  using S = Shape<N, HD>;
  static_assert(S::kBytes <= 232448, "shared memory");
  if (int st = allow_smem<k_tree_attention<DT, N, HD>>(S::kBytes)) return st;
  const int ctas = sm_count();
  const cudaError_t e = launch_ex(k_tree_attention<DT, N, HD>, dim3(ctas), dim3(kThreads), (size_t)S::kBytes, s, false, dim3(1), p);
  if (e != cudaSuccess) return fail(AF_ERR_CUDA, std::string("af_tree_attention: launch: ") + cudaGetErrorString(e));
  return join_launch<DT, N, HD>(p, ctas, s);
}

template <int DT, int HD>
int launch_rows(const Params& p, int n, cudaStream_t s) {
  return n == 16 ? launch<DT, 16, HD>(p, s) : n == 32 ? launch<DT, 32, HD>(p, s) : launch<DT, 64, HD>(p, s);
}

int launch_narrow(const Params& p, int n, bool bf16, int64_t head_dim, cudaStream_t s) {
  if (head_dim == 128) return bf16 ? launch_rows<AF_DTYPE_BF16, 128>(p, n, s) : launch_rows<AF_DTYPE_F16, 128>(p, n, s);
  return bf16 ? launch_rows<AF_DTYPE_BF16, 64>(p, n, s) : launch_rows<AF_DTYPE_F16, 64>(p, n, s);
}

}  // namespace

template <int DT, int N, int HD>
int join_launch(const Params& p, int ctas, cudaStream_t s) {
  if (p.capacity + p.total <= kWhole * kKeys) return check_launch("af_tree_attention");  // no row is shared
  const cudaError_t e = launch_ex(k_tree_attention_join<DT, N, HD>, dim3(ctas, kJoinBlocks<N>), dim3(kJoinThreads), 0, s, true, dim3(1), p, ctas);
  if (e != cudaSuccess) return fail(AF_ERR_CUDA, std::string("af_tree_attention: launch: ") + cudaGetErrorString(e));
  return check_launch("af_tree_attention");
}
template int join_launch<AF_DTYPE_F16, 256, 64>(const Params&, int, cudaStream_t);
template int join_launch<AF_DTYPE_F16, 256, 128>(const Params&, int, cudaStream_t);
template int join_launch<AF_DTYPE_BF16, 256, 64>(const Params&, int, cudaStream_t);
template int join_launch<AF_DTYPE_BF16, 256, 128>(const Params&, int, cudaStream_t);

}  // namespace tree_attn
}  // namespace af

using namespace af;
using namespace af::tree_attn;

extern "C" int af_tree_attention_workspace_bytes(int64_t* bytes) {
  AF_REQUIRE(bytes, "af_tree_attention_workspace_bytes: null pointer");
  *bytes = workspace_bytes();
  return AF_OK;
}

extern "C" int af_tree_attention_wait_limit(int64_t attempts) {
  AF_REQUIRE(attempts >= -1 && attempts <= kPatience, "af_tree_attention_wait_limit: attempts must lie between 0 and 2^18, or be -1");
  g_patience.store(attempts < 0 ? kPatience : (int)attempts, std::memory_order_relaxed);
  return AF_OK;
}

extern "C" int af_tree_attention(const af_tree_attention_args* args, uint32_t* status, void* stream) {
  AF_REQUIRE(args, "af_tree_attention: null pointer");
  const af_tree_attention_args& a = *args;
  if (int st = check_args(a)) return st;
  if (a.batch == 0 || a.total == 0) return AF_OK;
  Params p;
  memset(&p, 0, sizeof(p));
  const int group = (int)(a.n_heads / a.n_kv_heads);
  // Rows of a tile: the fewest that the average tree fits (the keys are read once per row tile); over 64 the wide kernel.
  const int64_t rows = ceil_div(a.total, a.batch) * group;
  const int n = rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 ? 64 : 256;
  const int box = (int)(a.page_size % 32 == 0 ? 32 : a.page_size % 16 == 0 ? 16 : 8);
  p.nt_q = (n == 256 ? 128 : n) / group;
  p.nt = n == 256 ? 2 * p.nt_q : p.nt_q;
  // Measured: a row end costs some 1800 cycles of 2700 a tile with 16 rows, 9000 of 2900 with 64, 8000 of 4500 with 256. With
  // 32 rows, 1 / 2 / 3 / 4 key tiles a row end: 32 requests of 28 rows over 300 to 4100 keys 56.7 / 55.2 / 53.9 / 52.4 us, 8
  // requests of 20 to 30 rows, 32 heads 92.3 / 91.4 / 82.7 / 72.8 us: 2 is low for them.
  p.row_cost = n == 16 ? 1 : n == 64 ? 3 : 2;
  // Tiles are counted in 32 bits: no more than this can come of any device-side values (starts out of order are refused there).
  AF_REQUIRE((double)a.n_kv_heads * (ceil_div(a.total, p.nt) + a.batch) * ((a.max_pages * a.page_size + a.total) / kKeys + 2 + p.row_cost) < 2147483000.0,
             "af_tree_attention: more than 2^31 tiles of 128 keys");
  const uint64_t hd = (uint64_t)a.head_dim, kvh = (uint64_t)a.n_kv_heads;
  {
    const uint64_t dims[3] = {hd, (uint64_t)a.n_heads, (uint64_t)a.total};
    const int64_t st[2] = {a.q_strides[1], a.q_strides[0]};
    const uint32_t bx[3] = {64, (uint32_t)group, (uint32_t)p.nt_q};
    if (int e = tree_map(&p.q, a.q, (int)a.dtype, 3, dims, st, bx)) return e;
  }
  for (int x = 0; x < 2; ++x) {
    const int64_t* rs = x ? a.v_strides : a.k_strides;
    const uint64_t dims[3] = {hd, kvh, (uint64_t)a.total};
    const int64_t st[2] = {rs[1], rs[0]};
    const uint32_t bx[3] = {64, 1, (uint32_t)box};
    if (int e = tree_map(x ? &p.v : &p.k, x ? a.v : a.k, (int)a.dtype, 3, dims, st, bx)) return e;
    if (a.pages == 0 || a.max_pages == 0) continue;
    const int64_t* cs = x ? a.v_cache_strides : a.k_cache_strides;
    const uint64_t cd[4] = {hd, kvh, (uint64_t)a.page_size, (uint64_t)a.pages};
    const int64_t ct[3] = {cs[2], cs[1], cs[0]};
    const uint32_t cb[4] = {64, 1, (uint32_t)box, 1};
    if (int e = tree_map(x ? &p.vc : &p.kc, x ? a.v_cache : a.k_cache, (int)a.dtype, 4, cd, ct, cb)) return e;
  }
  p.tables = a.tables;
  p.tables_ld = a.tables_stride;
  p.lengths = a.lengths;
  p.starts = a.starts;
  p.mask = reinterpret_cast<const uint32_t*>(a.mask);
  p.mask_ld = a.mask_stride;
  p.words = (int)a.words;
  p.batch = (int)a.batch;
  p.total = (int)a.total;
  p.kv_heads = (int)a.n_kv_heads;
  p.heads = (int)a.n_heads;
  p.group = group;
  p.pages = (int)a.pages;
  p.page = (int)a.page_size;
  p.box = box;
  p.capacity = a.pages ? a.max_pages * a.page_size : 0;
  p.scale = (float)(a.scale * 1.4426950408889634);
  p.v_rows = static_cast<const char*>(a.v);
  p.v_n = a.v_strides[0];
  p.v_h = a.v_strides[1];
  p.out = static_cast<char*>(a.out);
  p.out_n = a.out_strides[0];
  p.out_h = a.out_strides[1];
  p.lse = a.lse;
  p.ws = static_cast<char*>(a.workspace);
  p.status = status;
  p.patience = g_patience.load(std::memory_order_relaxed);
  cudaStream_t s = as_stream(stream);
  const bool bf16 = a.dtype == AF_DTYPE_BF16;
  return n == 256 ? wide_launch(p, bf16, (int)a.head_dim, s) : launch_narrow(p, n, bf16, a.head_dim, s);
}
