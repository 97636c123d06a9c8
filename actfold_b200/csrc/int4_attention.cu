// Attention of drafted trees over the 4-bit paged cache (sm_100a).
//
// With few rows per key/value head the work is one pass over the prefix's keys and
// values: 160 bytes a token and head of 128 dims, which become 256 values. At
// HBM's rate an SM has 7 cycles for those 256, so what a value costs on the way from its code
// to the product decides. Codes therefore go from shared memory straight into
// the registers of the warp-level products (m16n8k16), never through shared memory
// again as 16 bits, where writing and reading them would take up
// the SM's 128 bytes per cycle twice over (and tcgen05 takes its operands from there or from tensor memory):
//   S^T [16 keys, 8 rows] = K Q^T,       O^T [16 dims, 8 rows] += V^T P^T.
// Which dim or key an index of a fragment stands for is free as long as both operands agree,
// so a lane reads whole words: of K, for two keys, the 32 dims of one pair (16 bytes
// each); of V, for four keys, 16 dims (8 bytes each), two keys' half words put
// together before the codes are taken out. P^T gets from the accumulators' layout to the operand's by
// two 8 x 8 transposes.
//
// A producer warp plans (see int4_attention.cuh) and brings units of 32 keys, a bulk
// copy per page run, into a ring of slots; seven consumer warps take units in turn, each with maxima,
// sums and an O of its own, joined through shared memory at the end of a row tile. Up to 8 rows: two CTAs of 16 slots on an SM, whose
// ends of row tiles overlap (windows of 4100 tokens 160 -> 140 us); up to 16 rows: one CTA of 32 slots, for the registers. The step's own
// nodes are units too, read from their 16-bit rows. Every wait is bounded; a timeout sets AF_STATUS_TIMEOUT.
//
// No unit is near full: 0.52 to 0.59 instructions a cycle and scheduler, ALU pipe 45 %, HBM 35 to 40 %. What bounds it is a warp's chain
// through a unit (codes, values, products, softmax, products), some 860 instructions for 8 rows, of which the values take 512; the
// registers leave an SM 16 warps, too few to cover it. (A value is rounded once, as it is read back, which costs a subtraction and a
// multiply-add for each pair; scale and offset applied to sums of codes would need fewer, and give other scores. Not tried.)
// Probabilities are rounded to the values' type, which the products take (half a step of each; sums and outputs stay in 32 bits until
// the one rounding of the result): 0.0022 instead of 0.0017 over whole outputs in bf16, 0.00029 instead of 0.00021 in fp16.
//   64 requests of one token, 90 to 8000 keys, 28 heads over 4: 60 us; the bytes need 25.5.
//   24 requests of one token in windows of 4096 and 4 first tokens, 500 to 30000 keys, 32 heads over 32: 134 us; the bytes need 73.
//   One token over 523 keys: 10.9 us, of which a launch, the plan, a table, a unit and two joins are the chain.
// Tried: no producer, each warp brings its own units (spills); units by turns of 15 over two CTAs' warps (135 -> 150 us); Q of the
// next row tile ahead; 15 consumer warps in one CTA: slower or the same.
#include <math.h>

#include "int4_attention.cuh"

namespace af {

namespace kv4 {

namespace {

constexpr int kUnit = 32;    // keys of a unit

// NT: 8-row tiles of a warp; W: consumer warps; CTAS: on an SM.
template <int HD, int NT, int W, int CTAS>
struct Shape {
  static constexpr int kSlots = 32 / CTAS;
  static constexpr int kRows = 8 * NT;
  static constexpr int kUnitBytes = kUnit / kBlockTokens * Block<HD>::kBytes;
  static_assert(kSlots >= 16 && kSlots <= 32, "a producer fills eight at a time, others stay filled");
  static constexpr int kThreads = 32 * (W + 1);
  static constexpr int kOffAcc = kSlots * kUnitBytes;               // [W][kRows][HD] sums of the warps
  static constexpr int kOffStat = kOffAcc + W * kRows * HD * 4;     // [W][kRows] (maximum, sum)
  static constexpr int kOffBar = kOffStat + W * kRows * 8;
  static constexpr int kBars = 2 * kSlots + 2 * kPlans;
  static constexpr int kOffPlan = (kOffBar + 8 * kBars + 15) / 16 * 16;
  static constexpr int kBytes = kOffPlan + kPlans * (int)sizeof(Segment) + 16;
};

template <int DT>
__device__ __forceinline__ void mma(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (DT == AF_DTYPE_BF16) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  } else {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
}

__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

template <int BYTES>
__device__ __forceinline__ void lds(uint32_t at, uint32_t* r) {
  if constexpr (BYTES == 16)
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
  else if constexpr (BYTES == 8)
    asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(at) : "memory");
  else
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(r[0]) : "r"(at) : "memory");
}

__device__ __forceinline__ void bulk_copy(uint32_t dst, const char* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

// Plans the CTA's share, and brings its units of cached keys into the ring.
template <int HD, int NT, int W, int CTAS>
__device__ __forceinline__ void produce(const Params& p, uint8_t* gb, uint32_t base, uint32_t full, uint32_t empty, uint32_t plan_full,
                                        uint32_t plan_empty, Segment* plans, volatile int* failed) {
  using S = Shape<HD, NT, W, CTAS>;
  constexpr int kBlock = Block<HD>::kBytes, kSlots = S::kSlots;
  const int lane = threadIdx.x & 31;
  Planner<kUnit> planner;
  planner.begin(p, lane);
  Segment s;
  bool ok = true;
  int j = 0, issued = 0;  // units so far; the number behind the lane's last one
#pragma unroll 1
  for (int seg = 0; ok; ++seg) {
    const bool more = planner.next(p, s);
    if (seg >= kPlans) ok = __all_sync(0xffffffffu, wait_for(plan_empty + 8 * (seg % kPlans), (seg / kPlans - 1) & 1, failed));
    if (!ok) break;
    if (lane == 0) {
      plans[seg % kPlans] = s;
      mbar_arrive(plan_full + 8 * (seg % kPlans));
    }
    __syncwarp();
    if (!more) break;
    const int* table = p.tables + (int64_t)s.b * p.tables_ld;
    const char* head = p.data + s.kvh * p.d_head;
#pragma unroll 1
    for (int x0 = s.x0; ok && x0 < s.x1; x0 += 32) {
      // Lane x knows where unit x0 + x lies: the first run of blocks within a page, and the entries of the others.
      const int x = x0 + lane;
      const int place = kUnit * (x < s.sink_units ? x : x - s.sink_units + s.from);
      const int tokens = x < s.x1 && x < s.cached ? min(kUnit, s.len - place) : 0;
      const int all = (tokens + kBlockTokens - 1) / kBlockTokens;
      const int entry = tokens ? entry_of(p, place) : 0, at = (place - entry * p.page) / kBlockTokens;
      const int run = min(all, p.page / kBlockTokens - at);
      const int page = tokens ? table[entry] : 0;
      bool sound = page >= 0 && page < p.pages;
      const char* from = head + page * p.d_page + (int64_t)at * kBlock;
      const int me = j + lane, slot = me % kSlots;
      const uint32_t bar = full + 8 * slot, to = base + slot * S::kUnitBytes;
      const int count = min(32, s.x1 - x0);
      // Eight slots at a time, so that the others stay filled meanwhile.
#pragma unroll 1
      for (int i = 0; i < count; i += 8) {
        const bool mine = lane >= i && lane < min(count, i + 8);
        ok = __all_sync(0xffffffffu, !mine || me < kSlots || wait_for(empty + 8 * slot, (me / kSlots - 1) & 1, failed));
        if (!ok) break;
        if (mine) {
          if (all == 0) {
            mbar_arrive(bar);  // the step's own nodes: nothing to bring
          } else if (run == all && sound) {
            mbar_arrive_expect_tx(bar, all * kBlock);
            bulk_copy(to, from, all * kBlock, bar);
          } else {
            // Several pages, or one out of range, which reads as zeros.
            uint32_t bytes = 0;
            for (int y = 0, e = entry, n = run; y < all; y += n, ++e, n = min(all - y, p.page / kBlockTokens)) {
              const int pg = table[e];
              if (pg >= 0 && pg < p.pages) bytes += n * kBlock;
            }
            if (bytes < (uint32_t)(all * kBlock)) {
              if (p.status) atomicOr(p.status, AF_STATUS_BOUNDS);
              uint4* z = reinterpret_cast<uint4*>(gb + slot * S::kUnitBytes);
              for (int y = 0; y < S::kUnitBytes / 16; ++y) z[y] = make_uint4(0, 0, 0, 0);
              fence_proxy_async_smem();
            }
            mbar_arrive_expect_tx(bar, bytes);
            for (int y = 0, e = entry, n = run; y < all; y += n, ++e, n = min(all - y, p.page / kBlockTokens)) {
              const int pg = table[e];
              if (pg >= 0 && pg < p.pages) bulk_copy(to + y * kBlock, head + pg * p.d_page + (int64_t)(y ? 0 : at) * kBlock, n * kBlock, bar);
            }
          }
          issued = me + 1;
        }
        __syncwarp();
      }
      j += count;
    }
  }
  if (!ok) {
    *failed = 1;
    if (lane == 0 && p.status) atomicOr(p.status, AF_STATUS_TIMEOUT);
  }
  __syncwarp();
  // Copies still in flight (there are some only when a wait ran out) land before the CTA's shared memory is given up (bounded):
  // of the last kSlots units, one a lane.
  const int last = __reduce_max_sync(0xffffffffu, issued), mine = last - kSlots + lane;
  volatile int by_itself[2] = {0, kPatience};
  if (lane < kSlots && mine >= 0) wait_for(full + 8 * (mine % kSlots), (mine / kSlots) & 1, by_itself);
  __syncwarp();
}

template <int DT, int HD, int NT, int W, int CTAS>
__global__ void __launch_bounds__(32 * (W + 1), CTAS) k_int4_attention(const __grid_constant__ Params p) {
  using S = Shape<HD, NT, W, CTAS>;
  using B = Block<HD>;
  constexpr int kSlots = S::kSlots;
  constexpr int KW = HD / 32, KS = HD / 16;   // code words of a key that a lane takes; steps of the first product
  constexpr int VW = HD / 64, VT = HD / 16;   // code words of a value; 16-dim tiles of the second product
  constexpr int kTeam = 32 * W;
  extern __shared__ __align__(128) uint8_t gb[];
  pdl_trigger();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t base = smem_u32(gb);
  const uint32_t full = base + S::kOffBar, empty = full + 8 * kSlots, plan_full = empty + 8 * kSlots, plan_empty = plan_full + 8 * kPlans;
  Segment* plans = reinterpret_cast<Segment*>(gb + S::kOffPlan);
  volatile int* failed = reinterpret_cast<volatile int*>(gb + S::kOffPlan + kPlans * sizeof(Segment));
  if (tid == 0) {
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(full + 8 * i, 1);
      mbar_init(empty + 8 * i, 1);
    }
    for (int i = 0; i < kPlans; ++i) {
      mbar_init(plan_full + 8 * i, 1);
      mbar_init(plan_empty + 8 * i, W);
    }
    failed[0] = 0;
    failed[1] = p.patience;
    fence_barrier_init();
  }
  __syncthreads();
  const Scratch<S::kRows, HD> scratch{p.ws, (int)gridDim.x};

  if (warp == W) {
    produce<HD, NT, W, CTAS>(p, gb, base, full, empty, plan_full, plan_empty, plans, failed);
  } else {
    const int g = lane >> 2, t = lane & 3;
    // The key of a block that index g of the first product's M side stands for: indices 2 x and 2 x + 1, which a lane of the second
    // product takes together, are rows x and 4 + (x ^ 1), so that the rows that eight lanes read of K, and four of V, lie in different banks.
    const int kap = g & 1 ? 4 + ((g >> 1) ^ 1) : g >> 1;
    const uint32_t k_at = B::word(kap, KW * t), kp_at = B::pair(kap, (HD / 4) * t / kGroup);
    const uint32_t v_at0 = B::kPart + B::word(t, VW * g), v_at1 = B::kPart + B::word(4 + (t ^ 1), VW * g);
    const uint32_t vp_at0 = B::kPart + B::pair(t, (HD / 8) * g / kGroup), vp_at1 = B::kPart + B::pair(4 + (t ^ 1), (HD / 8) * g / kGroup);
    float* acc_all = reinterpret_cast<float*>(gb + S::kOffAcc);
    float2* stat_all = reinterpret_cast<float2*>(gb + S::kOffStat);
    int seg = 0;
    bool wrote_start = false;
    Segment s;
    // Into the next segment go all consumer warps or none, whatever each has seen of a plan or of a wait that ran out: the
    // barriers inside have no limit of their own. (It is also where the joins of the segment before are done with.)
    auto enter = [&]() {
      const bool there = __all_sync(0xffffffffu, wait_for(plan_full + 8 * (seg % kPlans), (seg / kPlans) & 1, failed));
      if (!there) *failed = 1;
      s = plans[seg % kPlans];
      __syncwarp();
      if (lane == 0) mbar_arrive(plan_empty + 8 * (seg % kPlans));
      return !vote_any<kTeam>(1, !there || s.x1 <= 0 || *failed);
    };
#pragma unroll 1
    while (enter()) {
      const int rows = min(S::kRows, s.n * p.group - s.row0);
      // Q: row 8 nt + g, the dims that this lane takes of a key.
      uint32_t q[NT][2 * KS];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int row = 8 * nt + g, flat = s.row0 + row;
        const char* at = p.q + (int64_t)(s.s0 + flat / p.group) * p.q_n + (s.kvh * p.group + flat % p.group) * p.q_h + t * (HD / 2);
#pragma unroll
        for (int i = 0; i < KS / 2; ++i) {
          const uint4 x = row < rows ? *reinterpret_cast<const uint4*>(at + 16 * i) : make_uint4(0, 0, 0, 0);
          // (p.scale is positive: the sign of the caller's goes to q, and 0 makes q 0)
          q[nt][4 * i] = (x.x ^ p.q_flip) & p.q_keep, q[nt][4 * i + 1] = (x.y ^ p.q_flip) & p.q_keep;
          q[nt][4 * i + 2] = (x.z ^ p.q_flip) & p.q_keep, q[nt][4 * i + 3] = (x.w ^ p.q_flip) & p.q_keep;
        }
      }
      // Rows 8 nt + 2 t and the next one: their nodes, and the first place of their windows.
      int node[NT][2], first[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          node[nt][e] = (s.row0 + min(8 * nt + 2 * t + e, rows - 1)) / p.group;
          first[nt][e] = first_place(p, s.s0, s.n, s.len, node[nt][e]);
        }
      // No row sees places from the sinks up to first_any; all see those from first_all on.
      const int first_any = p.window ? max(0, s.len - p.reach) : 0, first_all = p.window ? max(0, s.len - max(0, p.window - s.n)) : 0;
      float o[VT][NT][4];  // [dims 2 VT' .. of the lane's 16][row]
      float m[NT][2], l[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 2; ++e) m[nt][e] = kUnset, l[nt][e] = 0.f;
#pragma unroll
        for (int i = 0; i < VT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[i][nt][e] = 0.f;
      }
      // Scores of 16 keys (c: key g of their block 0, rows 2 t and 2 t + 1, then of block 1) into probabilities, the second product's
      // operand. seen(r, nt, e): does row e see key g of block r.
      auto softmax = [&](float (&x)[NT][4], uint32_t (&pf)[NT][2], bool masked, auto seen) {
        if (masked) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 4; ++c) x[nt][c] = seen(c >> 1, nt, c & 1) ? x[nt][c] : -INFINITY;
        }
        float top = -INFINITY;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) top = fmaxf(top, fmaf(fmaxf(x[nt][e], x[nt][2 + e]), p.scale, -m[nt][e]));
        if (__any_sync(0xffffffffu, top > kLead<DT> + kRaise)) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float y = fmaxf(x[nt][e], x[nt][2 + e]);
#pragma unroll
              for (int d = 4; d < 32; d <<= 1) y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, d));
              y *= p.scale;
              const float old = m[nt][e];
              if (old == kUnset ? y > kUnset : y > old + (kLead<DT> + kRaise)) {
                m[nt][e] = y - kLead<DT>;
                const float f = old == kUnset ? 0.f : exp2f(old - m[nt][e]);
                l[nt][e] *= f;
#pragma unroll
                for (int i = 0; i < VT; ++i) {
                  o[i][nt][e] *= f;
                  o[i][nt][2 + e] *= f;
                }
              }
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float y[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            y[c] = ex2(fmaf(x[nt][c], p.scale, -m[nt][c & 1]));
            l[nt][c & 1] += y[c];
          }
          pf[nt][0] = transposed(pack2<DT>(y[0], y[1]));
          pf[nt][1] = transposed(pack2<DT>(y[2], y[3]));
        }
      };
      const int x0 = s.x0 + (W + warp - s.j0 % W) % W;
#pragma unroll 1
      for (int x = x0; x < s.x1; x += W) {
        const int j = s.j0 + x - s.x0, slot = j % kSlots;
        if (!__all_sync(0xffffffffu, wait_for(full + 8 * slot, (j / kSlots) & 1, failed))) {
          *failed = 1;
          break;
        }
        if (x < s.cached) {
          // ---------------- 32 cached keys ----------------
          const int place = kUnit * (x < s.sink_units ? x : x - s.sink_units + s.from);
          const bool masked = place + kUnit > s.len || (p.window && place < first_all && place + kUnit > p.sinks);
          const uint32_t unit = base + slot * S::kUnitBytes;
          auto sees = [&](int at, int nt, int e) { return at < s.len && (at >= first[nt][e] || at < p.sinks); };
          bool sick = false;
          // S of both halves first: its chain of products is over by the time that the softmax looks at it.
          float both[2][NT][4];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t blocks = unit + 2 * h * B::kBytes;
            auto& sc = both[h];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int c = 0; c < 4; ++c) sc[nt][c] = 0.f;
            uint32_t w[2][KW], pr[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              lds<4 * KW>(blocks + r * B::kBytes + k_at, w[r]);
              lds<4>(blocks + r * B::kBytes + kp_at, &pr[r]);
            }
            const uint32_t s0 = __byte_perm(pr[0], 0, 0x1010), o0 = __byte_perm(pr[0], 0, 0x3232);
            const uint32_t s1 = __byte_perm(pr[1], 0, 0x1010), o1 = __byte_perm(pr[1], 0, 0x3232);
#pragma unroll
            for (int i = 0; i < KW; ++i) {
              const uint32_t a0 = two_values<DT, 0>(w[0][i], s0, o0), a1 = two_values<DT, 0>(w[1][i], s1, o1);
              const uint32_t a2 = two_values<DT, 1>(w[0][i], s0, o0), a3 = two_values<DT, 1>(w[1][i], s1, o1);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma<DT>(sc[nt], a0, a1, a2, a3, q[nt][4 * i], q[nt][4 * i + 1]);
              const uint32_t b0 = two_values<DT, 2>(w[0][i], s0, o0), b1 = two_values<DT, 2>(w[1][i], s1, o1);
              const uint32_t b2 = two_values<DT, 3>(w[0][i], s0, o0), b3 = two_values<DT, 3>(w[1][i], s1, o1);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma<DT>(sc[nt], b0, b1, b2, b3, q[nt][4 * i + 2], q[nt][4 * i + 3]);
            }
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t blocks = unit + 2 * h * B::kBytes;
            float sc[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int c = 0; c < 4; ++c) sc[nt][c] = h ? both[1][nt][c] : both[0][nt][c];
            uint32_t pf[NT][2];
            uint32_t w[2][2][VW], pr[2][2];  // [block][key of the lane's two]
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const uint32_t at = blocks + r * B::kBytes;
              lds<4 * VW>(at + v_at0, w[r][0]);
              lds<4 * VW>(at + v_at1, w[r][1]);
              lds<4>(at + vp_at0, &pr[r][0]);
              lds<4>(at + vp_at1, &pr[r][1]);
            }
            softmax(sc, pf, masked, [&](int r, int nt, int e) { return sees(place + 16 * h + 8 * r + kap, nt, e); });
            if (masked) {
              // What no row sees is 0 (behind the last token lies whatever was there); NaN that only some see is set aside.
#pragma unroll
              for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                  const int at = place + 16 * h + 8 * r + (b ? 4 + (t ^ 1) : t);
                  if (at >= s.len || (at < first_any && at >= p.sinks)) pr[r][b] = 0;
                  if (not_finite<DT>(pr[r][b] >> 16) || not_finite<DT>(pr[r][b])) {
                    sick = true;
                    pr[r][b] = 0;
                  }
                }
            }
            uint32_t s2[2], o2[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              s2[r] = __byte_perm(pr[r][0], pr[r][1], 0x5410);
              o2[r] = __byte_perm(pr[r][0], pr[r][1], 0x7632);
            }
#pragma unroll
            for (int i = 0; i < VW; ++i) {
              uint32_t lo[2], hi[2];  // the two keys' half words: codes of the even dims, and of the odd ones
#pragma unroll
              for (int r = 0; r < 2; ++r) {
                lo[r] = __byte_perm(w[r][0][i], w[r][1][i], 0x5410);
                hi[r] = __byte_perm(w[r][0][i], w[r][1][i], 0x7632);
              }
#define AF_STEP(I)                                                                                                                   \
  {                                                                                                                                  \
    const uint32_t a0 = two_values<DT, I>(lo[0], s2[0], o2[0]), a1 = two_values<DT, I>(hi[0], s2[0], o2[0]);                         \
    const uint32_t a2 = two_values<DT, I>(lo[1], s2[1], o2[1]), a3 = two_values<DT, I>(hi[1], s2[1], o2[1]);                         \
    _Pragma("unroll") for (int nt = 0; nt < NT; ++nt) mma<DT>(o[4 * i + I][nt], a0, a1, a2, a3, pf[nt][0], pf[nt][1]);               \
  }
              AF_STEP(0) AF_STEP(1) AF_STEP(2) AF_STEP(3)
#undef AF_STEP
            }
          }
          if (masked && __any_sync(0xffffffffu, sick)) {
            // Rare: a group of values that stands for NaN makes the dims of the rows that see it NaN.
#pragma unroll 1
            for (int y = 0; y < kUnit; ++y) {
              const int at = place + y;
              uint32_t pr;
              lds<4>(unit + y / kBlockTokens * B::kBytes + B::kPart + B::pair(y % kBlockTokens, (HD / 8) * g / kGroup), &pr);
              const bool bad = not_finite<DT>(pr >> 16) || not_finite<DT>(pr);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                  if (bad && sees(at, nt, e))
#pragma unroll
                    for (int i = 0; i < VT; ++i) o[i][nt][e] = o[i][nt][2 + e] = NAN;
            }
          }
        } else {
          // ---------------- 32 nodes of the tree, from their 16-bit rows ----------------
          const int j0 = kUnit * (x - s.cached);
          uint32_t bits[NT][2];
          uint32_t any = 0;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              bits[nt][e] = seen_nodes(p, s.s0, s.n, s.len, node[nt][e], j0);
              any |= bits[nt][e];
            }
          if (__any_sync(0xffffffffu, any != 0)) {  // (most units of a long chain are seen by no row of the tile)
            const char* k_row = p.k + (int64_t)s.s0 * p.k_n + s.kvh * p.k_h + t * (HD / 2);
            const char* v_row = p.v + (int64_t)s.s0 * p.v_n + s.kvh * p.v_h + g * (HD / 4);
            bool sick = false;
#pragma unroll 1
            for (int h = 0; h < 2; ++h) {
              if (j0 + 16 * h >= s.n) break;
              const int n0 = j0 + 16 * h + g, n1 = n0 + 8;
              float sc[NT][4];
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 4; ++c) sc[nt][c] = 0.f;
              uint32_t pf[NT][2];
#pragma unroll
              for (int i = 0; i < KS / 2; ++i) {
                const uint4 a = n0 < s.n ? *reinterpret_cast<const uint4*>(k_row + n0 * p.k_n + 16 * i) : make_uint4(0, 0, 0, 0);
                const uint4 b = n1 < s.n ? *reinterpret_cast<const uint4*>(k_row + n1 * p.k_n + 16 * i) : make_uint4(0, 0, 0, 0);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                  mma<DT>(sc[nt], a.x, b.x, a.y, b.y, q[nt][4 * i], q[nt][4 * i + 1]);
                  mma<DT>(sc[nt], a.z, b.z, a.w, b.w, q[nt][4 * i + 2], q[nt][4 * i + 3]);
                }
              }
              softmax(sc, pf, true, [&](int r, int nt, int e) { return ((bits[nt][e] >> (16 * h + 8 * r + g)) & 1u) != 0; });
#pragma unroll
              for (int i = 0; i < VT / 4; ++i) {
                uint32_t w[4][4];  // keys 2 t, 2 t + 1, and the same of the second block: 8 dims each
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                  const int at = j0 + 16 * h + 8 * (y >> 1) + 2 * t + (y & 1);
                  const uint4 a = at < s.n ? *reinterpret_cast<const uint4*>(v_row + at * p.v_n + 16 * i) : make_uint4(0, 0, 0, 0);
                  w[y][0] = a.x, w[y][1] = a.y, w[y][2] = a.z, w[y][3] = a.w;
#pragma unroll
                  for (int c = 0; c < 4; ++c) {
                    // A value that is not finite would reach every row as 0 * inf: it is set aside.
                    const bool lo = not_finite<DT>(w[y][c]), hi = not_finite<DT>(w[y][c] >> 16);
                    sick |= lo || hi;
                    w[y][c] &= (lo ? 0u : 0xffffu) | (hi ? 0u : 0xffff0000u);
                  }
                }
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                  const uint32_t a0 = __byte_perm(w[0][c], w[1][c], 0x5410), a1 = __byte_perm(w[0][c], w[1][c], 0x7632);
                  const uint32_t a2 = __byte_perm(w[2][c], w[3][c], 0x5410), a3 = __byte_perm(w[2][c], w[3][c], 0x7632);
#pragma unroll
                  for (int nt = 0; nt < NT; ++nt) mma<DT>(o[4 * i + c][nt], a0, a1, a2, a3, pf[nt][0], pf[nt][1]);
                }
              }
            }
            if (__any_sync(0xffffffffu, sick)) {
              // Rare: such values are added for the rows that see them.
#pragma unroll 1
              for (int y = 0; y < min(kUnit, s.n - j0); ++y) {
#pragma unroll
                for (int i = 0; i < VT; ++i) {
                  const uint32_t v2 = *reinterpret_cast<const uint32_t*>(v_row + (j0 + y) * p.v_n + 4 * i);
#pragma unroll
                  for (int d = 0; d < 2; ++d) {
                    const uint32_t b = d ? v2 >> 16 : v2 & 0xffffu;
                    if (not_finite<DT>(b)) {
#pragma unroll
                      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                          if ((bits[nt][e] >> y) & 1u) o[i][nt][2 * d + e] += from_bits<DT>(b);
                    }
                  }
                }
              }
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(empty + 8 * slot);
      }
      // ---------------- the warps' sums joined: row r, 16-byte pieces of 4 dims ----------------
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], d);
          if (g == 0) stat_all[warp * S::kRows + 8 * nt + 2 * t + e] = make_float2(m[nt][e], l[nt][e]);
        }
      named_bar_sync(1, kTeam);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int row = 8 * nt + 2 * t + e;
          float top = kUnset;
#pragma unroll
          for (int w = 0; w < W; ++w) top = fmaxf(top, stat_all[w * S::kRows + row].x);
          const float f = m[nt][e] == top ? 1.f : exp2f(m[nt][e] - top);
          // Dim 2 i + d of the lane's HD / 8; a row's pieces are exchanged by rows / 2, so that eight lanes write different banks.
          float* to = acc_all + (warp * S::kRows + row) * HD;
#pragma unroll
          for (int i = 0; i < VT / 2; ++i) {
            const int piece = (VT / 2) * g + i;
            *reinterpret_cast<float4*>(to + 4 * (piece ^ ((row >> 1) & 3))) =
                make_float4(o[2 * i][nt][e] * f, o[2 * i][nt][2 + e] * f, o[2 * i + 1][nt][e] * f, o[2 * i + 1][nt][2 + e] * f);
          }
        }
      named_bar_sync(1, kTeam);
      const bool whole = s.whole != 0;
      const int which = s.x0 == 0 ? 1 : 0;
#pragma unroll 1
      for (int item = tid; item < rows * (HD / 4); item += kTeam) {
        const int row = item / (HD / 4), piece = item % (HD / 4);
        float top = kUnset, sum = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) top = fmaxf(top, stat_all[w * S::kRows + row].x);
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < W; ++w) {
          const float2 ml = stat_all[w * S::kRows + row];
          sum += (ml.x == top ? 1.f : exp2f(ml.x - top)) * ml.y;
          const float4 a = *reinterpret_cast<const float4*>(acc_all + (w * S::kRows + row) * HD + 4 * (piece ^ ((row >> 1) & 3)));
          y.x += a.x, y.y += a.y, y.z += a.z, y.w += a.w;
        }
        if (whole) {
          const int flat = s.row0 + row, head = s.kvh * p.group + flat % p.group;
          const int64_t i = s.s0 + flat / p.group;
          const float inv = sum == 0.f ? 0.f : 1.f / sum;
          *reinterpret_cast<uint2*>(p.out + i * p.out_n + head * p.out_h + 8 * piece) = make_uint2(pack2<DT>(y.x * inv, y.y * inv), pack2<DT>(y.z * inv, y.w * inv));
          if (piece == 0 && p.lse) p.lse[i * p.heads + head] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
        } else {
          *reinterpret_cast<float4*>(scratch.sums(blockIdx.x, which) + row * HD + 4 * piece) = y;
          if (piece == 0) scratch.stats(blockIdx.x, which)[row] = make_float2(top, sum);
        }
      }
      if (!whole && s.x0 == 0) {
        wrote_start = true;
        if (tid == 0) *scratch.started(blockIdx.x) = Started{s.last, s.s0, s.row0, rows, s.kvh};
      }
      ++seg;
    }
    if (!wrote_start && tid == 0) scratch.started(blockIdx.x)->last = 0;
  }
  __syncthreads();
  if (tid == 0 && *failed && p.status) atomicOr(p.status, AF_STATUS_TIMEOUT);
}

template <int DT, int HD, int NT, int W, int CTAS>
int launch(const Params& p, cudaStream_t s) {
  using S = Shape<HD, NT, W, CTAS>;
  static_assert(CTAS * (S::kBytes + 1024) <= 233472, "shared memory");
  if (int st = allow_smem<k_int4_attention<DT, HD, NT, W, CTAS>>(S::kBytes, "af_tree_attention_int4")) return st;
  const int ctas = CTAS * sm_count();
  cudaError_t e = launch_ex(k_int4_attention<DT, HD, NT, W, CTAS>, dim3(ctas), dim3(S::kThreads), (size_t)S::kBytes, s, false, dim3(1), p);
  if (e == cudaSuccess && p.joins)
    e = launch_ex(k_join<DT, S::kRows, HD>, dim3(ctas, S::kRows), dim3(kJoinThreads), 0, s, true, dim3(1), p, ctas);
  if (e != cudaSuccess) return fail(AF_ERR_CUDA, std::string("af_tree_attention_int4: launch: ") + cudaGetErrorString(e));
  return check_launch("af_tree_attention_int4");
}

template <int DT, int HD>
int launch_rows(const Params& p, cudaStream_t s) {
  return p.rows == 8 ? launch<DT, HD, 1, 7, 2>(p, s) : launch<DT, HD, 2, 7, 1>(p, s);
}

int64_t workspace_bytes() { return Scratch<256, 128>::bytes(sm_count()); }

int check_args(const af_tree_attention_int4_args& a) {
  const af_int4_cache& c = a.cache;
  AF_REQUIRE(a.batch >= 0 && a.total >= 0 && a.max_pages >= 0 && c.pages >= 0, "af_tree_attention_int4: bad shape");
  AF_REQUIRE(a.n_heads > 0 && c.heads > 0 && a.n_heads % c.heads == 0, "af_tree_attention_int4: n_heads must be a multiple of the cache's heads");
  AF_REQUIRE(c.head_dim == 64 || c.head_dim == 128, "af_tree_attention_int4: head_dim must be 64 or 128");
  AF_REQUIRE(c.dtype == AF_DTYPE_F16 || c.dtype == AF_DTYPE_BF16, "af_tree_attention_int4: dtype must be fp16 or bf16");
  AF_REQUIRE(c.page_size > 0 && c.page_size % kBlockTokens == 0 && c.page_size <= (1 << 20), "af_tree_attention_int4: page_size must be a multiple of 8");
  AF_REQUIRE(a.batch <= AF_TREE_ATTN_MAX_BATCH, "af_tree_attention_int4: at most 16384 requests");
  AF_REQUIRE(a.total <= (1 << 28) && c.pages <= 0x7fffffff && a.n_heads <= (1 << 16) && a.max_pages <= (1 << 30) && a.max_pages * c.page_size <= (1 << 30) &&
                 a.total * (a.n_heads / c.heads) <= (1 << 30),
             "af_tree_attention_int4: size too large");
  AF_REQUIRE(a.window >= 0 && a.sinks >= 0 && a.window <= (1 << 30) && a.sinks <= (1 << 30), "af_tree_attention_int4: window and sinks must not be negative");
  AF_REQUIRE(!a.mask || (a.words > 0 && a.words <= AF_TREE_MAX_NODES / 32 && a.mask_stride >= a.words), "af_tree_attention_int4: bad mask");
  if (a.batch == 0 || a.total == 0) return AF_OK;
  AF_REQUIRE(runs_apart(c, false), "af_tree_attention_int4: the cache's strides let its entries share memory");
  AF_REQUIRE(a.q && a.k && a.v && a.out && a.lengths && a.starts && a.workspace, "af_tree_attention_int4: null pointer");
  AF_REQUIRE(a.max_pages == 0 || c.pages == 0 || (c.data && a.tables), "af_tree_attention_int4: null pointer");
  uint64_t al = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v) |
                reinterpret_cast<uintptr_t>(c.data) | reinterpret_cast<uintptr_t>(a.out) | reinterpret_cast<uintptr_t>(a.workspace);
  for (int i = 0; i < 2; ++i)
    al |= (uint64_t)a.q_strides[i] | (uint64_t)a.k_strides[i] | (uint64_t)a.v_strides[i] | (uint64_t)a.out_strides[i];
  for (int i = 1; i < 3; ++i) al |= (uint64_t)c.strides[i];
  AF_REQUIRE((al & 15) == 0, "af_tree_attention_int4: addresses and strides must be multiples of 16 bytes");
  AF_REQUIRE(a.workspace_bytes >= workspace_bytes(), "af_tree_attention_int4: the workspace is too small");
  return AF_OK;
}

}  // namespace
}  // namespace kv4
}  // namespace af

using namespace af;

extern "C" int af_tree_attention_int4_workspace_bytes(int64_t* bytes) {
  AF_REQUIRE(bytes, "af_tree_attention_int4_workspace_bytes: null pointer");
  *bytes = kv4::workspace_bytes();
  return AF_OK;
}

extern "C" int af_tree_attention_int4(const af_tree_attention_int4_args* args, uint32_t* status, void* stream) {
  AF_REQUIRE(args, "af_tree_attention_int4: null pointer");
  const af_tree_attention_int4_args& a = *args;
  const af_int4_cache& c = a.cache;
  if (int st = kv4::check_args(a)) return st;
  if (a.batch == 0 || a.total == 0) return AF_OK;
  kv4::Params p;
  memset(&p, 0, sizeof(p));
  p.q = static_cast<const char*>(a.q), p.q_n = a.q_strides[0], p.q_h = a.q_strides[1];
  p.k = static_cast<const char*>(a.k), p.k_n = a.k_strides[0], p.k_h = a.k_strides[1];
  p.v = static_cast<const char*>(a.v), p.v_n = a.v_strides[0], p.v_h = a.v_strides[1];
  p.data = static_cast<const char*>(c.data), p.d_page = c.strides[1], p.d_head = c.strides[2];
  p.tables = a.tables;
  p.tables_ld = a.tables_stride;
  p.lengths = a.lengths;
  p.starts = a.starts;
  p.mask = reinterpret_cast<const uint32_t*>(a.mask);
  p.mask_ld = a.mask_stride;
  p.words = (int)a.words;
  p.batch = (int)a.batch;
  p.total = (int)a.total;
  p.heads = (int)a.n_heads;
  p.kv_heads = (int)c.heads;
  p.group = (int)(a.n_heads / c.heads);
  p.pages = (int)c.pages;
  kv4::set_page(p, c.page_size);
  p.capacity = c.pages ? a.max_pages * c.page_size : 0;
  p.window = (int)a.window;
  p.sinks = (int)a.sinks;
  p.reach = p.window - (a.mask ? 0 : 1);
  p.scale = (float)(fabs(a.scale) * 1.4426950408889634);
  p.q_flip = a.scale < 0. ? 0x80008000u : 0u;
  p.q_keep = p.scale == 0.f ? 0u : 0xffffffffu;
  if (p.scale == 0.f) p.scale = 1.f;  // (0, and what is 0 in fp32: hidden scores of -inf times 0 would be NaN)
  p.out = static_cast<char*>(a.out), p.out_n = a.out_strides[0], p.out_h = a.out_strides[1];
  p.lse = a.lse;
  p.ws = static_cast<char*>(a.workspace);
  p.status = status;
  p.patience = attention_patience();
  // Rows of the average request and head choose the kernel and its row tile. 16 requests of 300 to 4100 keys, 4 heads of keys:
  //   12 and 16 rows: 28.4 and 29.3 us in one tile of 16, 29.6 and 30.2 in two of 8, 32.7 and 32.8 as 128 (tensor cores);
  //   20 and 28 rows: 35.4 and 36.4 us in two tiles of 16, 33.5 and 33.8 as 128;
  //   140 and 224 rows: 50.5 and 57.0 us as 256, 56.0 and 61.3 in two tiles of 128.
  const int64_t rows = ceil_div(a.total, a.batch) * p.group;
  const bool wide = rows > 16;
  p.rows = rows <= 8 ? 8 : rows <= 16 ? 16 : rows <= 128 ? 128 : 256;
  // What a row tile costs besides its units (of 32 keys; wide 128), in units: the joins of the warps, the output. Few rows: 64 tokens
  // 63.6 us with 4, 60.5 with 10, 59.4 with 20, but where few rows are cut into more (8 requests of up to 1500 keys, 32 heads) 31.8, 27.5, 30.6. Wide:
  // 8 trees 111 us with 1, 94 with 3, 96 with 8; 2 of 64 nodes over 30000 keys, two row tiles, 120 with 1, 110 with 5 and 8.
  p.row_cost = p.rows > 128 ? 5 : wide ? 3 : 10;
  // Units up to which a row tile is not cut: a second CTA's part costs a trip through memory and the join. One token over 523 keys
  // 10.4 us with 32, 13.0 with 8; where shares are long such rows would make them uneven: 64 tokens 60.5 us with 8, 67.7 with 32.
  // Wide: 16 requests of 21 to 42 rows 34 us with 2, 46 with 8.
  p.whole = wide ? 2 : 32;
  p.whole_long = wide ? 2 : 8;
  // Units of a share, at least. Few rows: one token over 2000 and up to 8000 keys 13.7 and 14.9 us with 14, 17.2 and 18.5 with 28, 13.1
  // and 15.8 with 4. Wide: one tree of 26 nodes over 900 keys 25.7 us with 2, 30.5 with 1, 34.7 with 6.
  p.least = wide ? 2 : 14;
  // Units are counted in 32 bits: no more than this can come of any device-side values (starts out of order are refused there).
  const int64_t most = (a.max_pages * c.page_size + a.total) / (wide ? kv4::kWideUnit : kv4::kUnit) + 3;  // of a row tile
  const double all = (double)c.heads * (ceil_div(a.total * p.group, p.rows) + a.batch) * (most + p.row_cost);
  AF_REQUIRE(all < 2147483000.0, "af_tree_attention_int4: more than 2^31 units of keys");
  p.joins = most > (all >= 2.0 * p.whole * sm_count() ? p.whole_long : p.whole);
  cudaStream_t s = as_stream(stream);
  const bool bf16 = c.dtype == AF_DTYPE_BF16;
  if (wide) return kv4::wide_launch(p, bf16, (int)c.head_dim, s);
  if (c.head_dim == 128) return bf16 ? kv4::launch_rows<AF_DTYPE_BF16, 128>(p, s) : kv4::launch_rows<AF_DTYPE_F16, 128>(p, s);
  return bf16 ? kv4::launch_rows<AF_DTYPE_BF16, 64>(p, s) : kv4::launch_rows<AF_DTYPE_F16, 64>(p, s);
}
