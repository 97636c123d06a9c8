// Attention of drafted trees over a paged key/value cache (sm_100a, tcgen05).
//
// For every request and key/value head, the rows (node, query head of the
// group) of its tree attend to the cached prefix and to the visible nodes of
// the tree. With few rows per head the work is one pass over the prefix's
// keys and values, so the products are transposed: the 128 KEYS of a tile are
// the M side of the tensor-core instruction and the rows (64 or 128 of them)
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
// Warps 0-7 run the softmax (warp w: TMEM lanes 32 (w & 3).. = keys, columns
// of half w >> 2), warp 8 loads (TMA), warp 9 issues the products. A column's
// reference maximum m is raised only when a score passes it by more than 2^8
// (or at the row's first key): steady tiles take one comparison per score and one
// barrier vote, no maximum across lanes. P then stays below 256, which bf16
// and fp16 round with the same relative error. Sums and O are fp32. Every wait is
// bounded; a timeout sets AF_STATUS_TIMEOUT.
#include <cuda.h>

#include "tree.cuh"

namespace af {

namespace {

constexpr int kKeys = 128;                  // keys per tile (MMA M)
constexpr int kHalf = kKeys * 128;          // [128 rows][64 columns] of 16 bits, 128-byte swizzle
constexpr int kSoft = 8;                    // softmax warps
constexpr int kThreads = (kSoft + 2) * 32;
constexpr float kUnset = -3.0e38f;          // reference maximum of a row that has seen no key
constexpr float kRaise = 8.f;               // log2 headroom before a reference maximum is raised

// Shared memory: stages of (K, V) tiles, Q, and a little state. P^T of a tile
// goes over its keys, which nobody needs once S is there.
template <int N, int HD>
struct Shape {
  static constexpr int kHalves = HD / 64;
  static constexpr int kPBytes = (N / 64) * kHalf;  // [128 keys][64 rows] blocks
  static constexpr int kKBytes = kHalves * kHalf > kPBytes ? kHalves * kHalf : kPBytes;
  static constexpr int kStage = kKBytes + kHalves * kHalf;
  static constexpr int kStages = (192 * 1024) / kStage;
  static constexpr int kQBytes = kHalves * N * 128;
  static constexpr int kQ = kQBytes <= 16384 ? 2 : 1;         // Q buffers
  static constexpr int kOffQ = kStages * kStage;
  static constexpr int kOffM = kOffQ + kQ * kQBytes;          // [N] reference maxima
  static constexpr int kOffRed = kOffM + N * 4;               // [4][N] per-warp maxima or sums; row 0: factors, row sums
  static constexpr int kOffBar = kOffRed + 4 * N * 4;
  static constexpr int kBytes = kOffBar + 384;
};

struct Params {
  CUtensorMap q, k, v, kc, vc;
  const int *tables, *lengths, *starts;
  const uint32_t* mask;
  int64_t tables_ld, mask_ld;
  int words, batch, total, kv_heads, group, pages, page, box, nt;
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
};

// A request's tree and prefix; tiles = 0 where there is nothing to do or the values are bad.
struct Request {
  int s0, n, len, pad, kt, qt;
  bool bad;
  __device__ __forceinline__ int64_t tiles(int kv_heads) const { return (int64_t)kt * qt * kv_heads; }
};

__device__ __forceinline__ Request request(const Params& p, int b) {
  Request r;
  const int s0 = p.starts[b], s1 = p.starts[b + 1];
  r.len = p.lengths[b];
  r.bad = s0 < 0 || s1 < s0 || s1 > p.total || r.len < 0 || r.len > p.capacity || (p.mask && s1 - s0 > 32 * (int64_t)p.words);
  r.s0 = s0;
  r.n = r.bad ? 0 : s1 - s0;
  r.pad = (r.len + p.box - 1) / p.box * p.box;
  r.kt = r.n ? (int)(((int64_t)r.pad + r.n + kKeys - 1) / kKeys) : 0;
  r.qt = (r.n + p.nt - 1) / p.nt;
  return r;
}

// The tiles [k0, k1) of one row tile that a CTA works on.
struct Segment {
  Request r;
  int kvh, qt, k0, k1;
  int64_t row_end;  // list index behind the row tile's last tile
  __device__ __forceinline__ bool whole() const { return k0 == 0 && k1 == r.kt; }
};

struct Walk {
  int64_t t, end, before;  // next tile, last one, tiles of the requests before b
  int b;
  __device__ __forceinline__ bool next(const Params& p, Segment& s) {
    if (t >= end) return false;
    s.r = request(p, b);
    while (t >= before + s.r.tiles(p.kv_heads)) {
      before += s.r.tiles(p.kv_heads);
      s.r = request(p, ++b);
    }
    const int64_t rel = t - before;
    const int64_t row = rel / s.r.kt;
    s.k0 = (int)(rel - row * s.r.kt);
    s.k1 = (int)min((int64_t)s.r.kt, s.k0 + (end - t));
    s.qt = (int)(row % s.r.qt);
    s.kvh = (int)(row / s.r.qt);
    s.row_end = before + (row + 1) * s.r.kt;
    t += s.k1 - s.k0;
    return true;
  }
};

// What CTA c left for k_tree_attention_join: it began a row tile that CTAs
// c + 1 .. last went on with (last = 0: it did not).
struct Started {
  int last, node0, rows, kvh;
};

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

__device__ __forceinline__ float ex2(float x) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x));
  return e;
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

__device__ __forceinline__ void tmem_store32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}

// 32 values per lane reduced across the warp: lane j returns the result of
// values j. Each step halves the values that a lane keeps (31 exchanges, where
// a reduction per value takes 160).
template <typename Op>
__device__ __forceinline__ float transpose_reduce(float* v, int lane, Op op) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const bool up = (lane & o) != 0;
#pragma unroll
    for (int i = 0; i < o; ++i) {
      const float give = up ? v[i] : v[i + o], keep = up ? v[i + o] : v[i];
      v[i] = op(keep, __shfl_xor_sync(0xffffffffu, give, o));
    }
  }
  return v[0];
}

// Bits of the warp's 32 keys (nodes j0, j0 + 1, ... of the tree) that node i
// sees; a bit outside the tree means nothing.
__device__ __forceinline__ uint32_t seen_bits(const Params& p, const Segment& s, int i, int j0) {
  if (!p.mask) return i < j0 ? 0u : i - j0 >= 31 ? 0xffffffffu : (2u << (i - j0)) - 1u;
  const uint32_t* row = p.mask + (int64_t)(s.r.s0 + i) * p.mask_ld;
  const int w = j0 >> 5;  // j0 may be negative: rounds down
  const uint32_t lo = w >= 0 && w < p.words ? row[w] : 0u, hi = w + 1 >= 0 && w + 1 < p.words ? row[w + 1] : 0u;
  return __funnelshift_r(lo, hi, j0 & 31);
}

template <int DT, int N, int HD>
__global__ void __launch_bounds__(kThreads, 1) k_tree_attention(const __grid_constant__ Params p) {
  using S = Shape<N, HD>;
  extern __shared__ __align__(1024) uint8_t gb[];
  pdl_trigger();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t base = smem_u32(gb), sQ = base + S::kOffQ;
  auto sK = [&](int stage) { return base + stage * S::kStage; };
  auto sV = [&](int stage) { return base + stage * S::kStage + S::kKBytes; };
  // K full, V full, stage empty [stages]; then pairs: Q full, Q empty, S full, P full, O of a tile done, O full, O empty
  const uint32_t k_full = base + S::kOffBar, v_full = k_full + 8 * S::kStages, empty = v_full + 8 * S::kStages,
                 q_full = empty + 8 * S::kStages, q_empty = q_full + 16, s_full = q_empty + 16, p_full = s_full + 16,
                 done = p_full + 16, o_full = done + 16, o_empty = o_full + 16;
  static_assert(24 * S::kStages + 7 * 16 <= 256, "barriers");
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(gb + S::kOffBar + 256);
  volatile int* failed = reinterpret_cast<volatile int*>(gb + S::kOffBar + 260);
  int* found_b = reinterpret_cast<int*>(gb + S::kOffBar + 264);
  int64_t* found = reinterpret_cast<int64_t*>(gb + S::kOffBar + 272);  // tiles before request found_b
  int64_t* scan = reinterpret_cast<int64_t*>(gb + S::kOffBar + 280);   // sums of the warps
  static_assert(280 + 8 * kThreads / 32 <= 384, "scan");

  if (tid == 0) {
    for (int i = 0; i < S::kStages; ++i) {
      mbar_init(k_full + 8 * i, 1);
      mbar_init(v_full + 8 * i, 1);
      mbar_init(empty + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(q_full + 8 * i, 1);
      mbar_init(q_empty + 8 * i, 1);
      mbar_init(s_full + 8 * i, 1);
      mbar_init(p_full + 8 * i, kSoft);
      mbar_init(done + 8 * i, 1);
      mbar_init(o_full + 8 * i, 1);
      mbar_init(o_empty + 8 * i, kSoft);
    }
    *failed = 0;
    fence_barrier_init();
  }
  if (warp == kSoft) tmem_alloc(smem_u32(tmem_slot), 4 * N);

  // This CTA's share [t0, t1) of the list of tiles, and the request it begins with.
  const int per = (p.batch + kThreads - 1) / kThreads, b_lo = min(p.batch, tid * per), b_hi = min(p.batch, b_lo + per);
  int64_t mine = 0;
  for (int b = b_lo; b < b_hi; ++b) {
    const Request r = request(p, b);
    mine += r.tiles(p.kv_heads);
    if (r.bad && blockIdx.x == 0 && p.status) atomicOr(p.status, AF_STATUS_BOUNDS);
  }
  int64_t upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += y;
  }
  if (lane == 31) scan[warp] = upto;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  int64_t all = 0, at = upto - mine;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) at += scan[w];
    all += scan[w];
  }
  const int64_t ctas = min((int64_t)gridDim.x, all);
  const int64_t t0 = blockIdx.x < ctas ? all * blockIdx.x / ctas : 0, t1 = blockIdx.x < ctas ? all * (blockIdx.x + 1) / ctas : 0;
  if (t0 < t1 && at <= t0 && t0 < at + mine) {
    for (int b = b_lo; b < b_hi; ++b) {
      const int64_t w = request(p, b).tiles(p.kv_heads);
      if (t0 < at + w) {
        *found_b = b;
        *found = at;
        break;
      }
      at += w;
    }
  }
  __syncthreads();
  const uint32_t tmem = *tmem_slot;
  const Scratch<N, HD> scratch{p.ws, (int)gridDim.x};
  Walk walk;
  walk.t = t0;
  walk.end = t1;
  walk.b = t0 < t1 ? *found_b : 0;
  walk.before = t0 < t1 ? *found : 0;
  Segment s;

  if (warp == kSoft) {
    // ---------------- loads: Q of a segment, then K and V of its tiles into the stages ----------------
    const int boxes = kKeys / p.box;
    int j = 0, seg = 0;
    bool ok = true;
    while (ok && walk.next(p, s)) {
      const int qb = seg % S::kQ, use = seg / S::kQ;
      if (use > 0) ok = mbar_wait(q_empty + 8 * qb, (use - 1) & 1, failed);
      if (!ok) break;
      if (lane == 0) {
        mbar_arrive_expect_tx(q_full + 8 * qb, S::kHalves * p.nt * p.group * 128);
        for (int h = 0; h < S::kHalves; ++h)
          tma_load_3d(sQ + qb * S::kQBytes + h * N * 128, &p.q, q_full + 8 * qb, 64 * h, s.kvh * p.group, s.r.s0 + s.qt * p.nt);
      }
      ++seg;
      // Lane (box, half) loads rows [box * R, (box + 1) * R) of each tile; the page is fetched a tile ahead.
      const int box = lane / S::kHalves, half = lane % S::kHalves, row = box * p.box;
      const int* table = p.tables + (int64_t)walk.b * p.tables_ld;
      auto page_of = [&](int kt) {
        const int key = kt * kKeys + row;
        return box < boxes && kt < s.k1 && key < s.r.len ? table[key / p.page] : 0;
      };
      int page = page_of(s.k0);
      for (int kt = s.k0; kt < s.k1; ++kt, ++j) {
        const int key = kt * kKeys + row;
        const int node = key - s.r.pad;
        const bool cached = box < boxes && key < s.r.len, tree = box < boxes && node >= 0 && node < s.r.n;
        if (cached && (page < 0 || page >= p.pages)) {
          if (p.status) atomicOr(p.status, AF_STATUS_BOUNDS);
          page = p.pages;  // out of range: the box reads as zeros
        }
        const unsigned who = __ballot_sync(0xffffffffu, cached || tree);
        const uint32_t bytes = __popc(who) * p.box * 128;
        const int off = cached ? key % p.page : 0;
        const int stage = j % S::kStages, round = j / S::kStages;
        if (round > 0) ok = mbar_wait(empty + 8 * stage, (round - 1) & 1, failed);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (lane == 0) {
          mbar_arrive_expect_tx(k_full + 8 * stage, bytes);
          mbar_arrive_expect_tx(v_full + 8 * stage, bytes);
        }
        __syncwarp();
        const uint32_t at = half * kHalf + row * 128;
        if (cached) {
          tma_load_4d(sK(stage) + at, &p.kc, k_full + 8 * stage, 64 * half, s.kvh, off, page);
          tma_load_4d(sV(stage) + at, &p.vc, v_full + 8 * stage, 64 * half, s.kvh, off, page);
        } else if (tree) {
          tma_load_3d(sK(stage) + at, &p.k, k_full + 8 * stage, 64 * half, s.kvh, s.r.s0 + node);
          tma_load_3d(sV(stage) + at, &p.v, v_full + 8 * stage, 64 * half, s.kvh, s.r.s0 + node);
        }
        page = page_of(kt + 1);
      }
    }
    if (!ok) {
      *failed = 1;
      if (lane == 0 && p.status) atomicOr(p.status, AF_STATUS_TIMEOUT);
    }
    __syncwarp();
    if (*failed && lane == 0) {
      // Copies still in flight land before the CTA's shared memory is given up (bounded).
      volatile int no_abort = 0;
      for (int i = max(0, j - S::kStages); i < j; ++i) {
        mbar_wait(k_full + 8 * (i % S::kStages), (i / S::kStages) & 1, &no_abort);
        mbar_wait(v_full + 8 * (i % S::kStages), (i / S::kStages) & 1, &no_abort);
      }
      for (int i = max(0, seg - S::kQ); i < seg; ++i) mbar_wait(q_full + 8 * (i % S::kQ), (i / S::kQ) & 1, &no_abort);
    }
  } else if (warp == kSoft + 1 && lane == 0) {
    // ---------------- products: S_j, then O += V P of tile j - 1 ----------------
    constexpr uint32_t kind = DT == AF_DTYPE_BF16 ? 0u : ((1u << 7) | (1u << 10));  // formats: bf16 = 1, f16 = 0
    constexpr uint32_t id_s = idesc_bf16(kKeys, N) ^ kind;
    constexpr uint32_t id_o = (idesc_bf16(128, N) ^ kind) | (1u << 15) | (1u << 16);  // A and B MN-major
    bool ok = true;
    int j = 0, seg = 0;
    // State of tile j - 1 for its second product.
    int last_seg = 0;
    bool last_first = false, last_last = false;
    auto second = [&](int i) {
      const int pb = i & 1, stage = i % S::kStages, ob = last_seg & 1;
      ok = mbar_wait(p_full + 8 * pb, (i >> 1) & 1, failed) && mbar_wait(v_full + 8 * stage, (i / S::kStages) & 1, failed);
      if (ok && last_first && last_seg >= 2) ok = mbar_wait(o_empty + 8 * ob, ((last_seg >> 1) - 1) & 1, failed);
      if (!ok) return;
      tc_fence_after();
#pragma unroll
      for (int kk = 0; kk < kKeys / 16; ++kk) {
        const uint64_t a = sw128_desc_mn(sV(stage) + kk * 2048, kHalf, 1024);
        const uint64_t b = sw128_desc_mn(sK(stage) + kk * 2048, kHalf, 1024);
        tc_mma_bf16(tmem + 2 * N + ob * N, a, b, id_o, last_first && kk == 0 ? 0u : 1u);
      }
      tc_commit(empty + 8 * stage);
      tc_commit(done + 8 * pb);
      if (last_last) tc_commit(o_full + 8 * ob);
    };
    while (ok && walk.next(p, s)) {
      const int qb = seg % S::kQ;
      for (int kt = s.k0; ok && kt < s.k1; ++kt, ++j) {
        const int sb = j & 1, stage = j % S::kStages;
        // With one Q buffer the next rows arrive after the last S of these ones: do what is left first.
        const bool early = S::kQ == 1 && kt == s.k0 && j > 0;
        if (early) second(j - 1);
        if (ok && kt == s.k0) ok = mbar_wait(q_full + 8 * qb, (seg / S::kQ) & 1, failed);
        ok = ok && mbar_wait(k_full + 8 * stage, (j / S::kStages) & 1, failed);
        // S buffer sb is read: P of tile j - 2 was waited for by its second product.
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk) {
          const uint64_t a = sw128_desc(sK(stage) + (kk >> 2) * kHalf) + 2 * (kk & 3);
          const uint64_t b = sw128_desc(sQ + qb * S::kQBytes + (kk >> 2) * N * 128) + 2 * (kk & 3);
          tc_mma_bf16(tmem + sb * N, a, b, id_s, kk ? 1u : 0u);
        }
        tc_commit(s_full + 8 * sb);
        if (kt + 1 == s.k1) tc_commit(q_empty + 8 * qb);
        if (j > 0 && !early) second(j - 1);
        last_seg = seg;
        last_first = kt == s.k0;
        last_last = kt + 1 == s.k1;
      }
      ++seg;
    }
    if (ok && j > 0) second(j - 1);
    if (!ok) {
      *failed = 1;
      if (p.status) atomicOr(p.status, AF_STATUS_TIMEOUT);
    }
  } else if (warp < kSoft) {
    // ---------------- softmax: key 32 * quad + lane, columns c0 .. c0 + C - 1 ----------------
    constexpr int C = N / 2, G32 = C / 32;
    const int quad = warp & 3, wg = warp >> 2, r = 32 * quad + lane, c0 = wg * C, wg_tid = tid - 128 * wg;
    const uint32_t lanes = tmem + ((uint32_t)(32 * quad) << 16);
    float* m_ref = reinterpret_cast<float*>(gb + S::kOffM) + c0;
    float* red = reinterpret_cast<float*>(gb + S::kOffRed) + c0;  // red[w * N + column]
    float* factor = red;
    auto wait = [&](uint32_t bar, uint32_t parity) {
      if (!mbar_wait(bar, parity, failed)) *failed = 1;
    };
    int j = 0, seg = 0;
    bool wrote_start = false;
    while (walk.next(p, s)) {
      const int nodes = min(p.nt, s.r.n - s.qt * p.nt), cols = nodes * p.group;
      const int live = min(C, max(0, cols - c0));  // columns of this half that are rows
      float l[C];
#pragma unroll
      for (int i = 0; i < C; ++i) l[i] = 0.f;
      if (wg_tid < C) m_ref[wg_tid] = kUnset;
      bool sick = false;  // a visible value that is not finite was set aside
      named_bar_sync(1 + wg, 128);
      for (int kt = s.k0; kt < s.k1; ++kt, ++j) {
        const int sb = j & 1, stage = j % S::kStages, key0 = kt * kKeys, key = key0 + r;
        const bool masked = key0 + kKeys > s.r.len;
        uint32_t vis[G32];
        if (masked) {
          const int node = key - s.r.pad, j0 = key0 + 32 * quad - s.r.pad;
          const bool in_prefix = key < s.r.len, in_tree = node >= 0 && node < s.r.n;
#pragma unroll
          for (int g = 0; g < G32; ++g) {
            const int c = c0 + 32 * g + lane;
            const uint32_t bits = c < cols ? seen_bits(p, s, s.qt * p.nt + c / p.group, j0) : 0u;
            uint32_t v = 0;
#pragma unroll
            for (int i = 0; i < 32; ++i) v |= ((__shfl_sync(0xffffffffu, bits, i) >> lane) & 1u) << i;
            vis[g] = in_prefix ? 0xffffffffu : in_tree ? v : 0u;
          }
        }
        wait(s_full + 8 * sb, (j >> 1) & 1);
        tc_fence_after();
        uint32_t x[C];
        auto load_scores = [&]() {
#pragma unroll
          for (int g = 0; g < G32; ++g)
            if (32 * g < live) tmem_ld32_nowait(lanes + sb * N + c0 + 32 * g, x + 32 * g);
          tmem_wait_ld();
        };
        load_scores();
        // x = score - reference maximum (in log2 units); hidden scores -inf.
        float top = -INFINITY;
        auto shift = [&]() {
#pragma unroll
          for (int q8 = 0; q8 < C / 8; ++q8) {
            if (8 * q8 < live) {
              const float4 m0 = *reinterpret_cast<const float4*>(m_ref + 8 * q8), m1 = *reinterpret_cast<const float4*>(m_ref + 8 * q8 + 4);
              const float mm[8] = {m0.x, m0.y, m0.z, m0.w, m1.x, m1.y, m1.z, m1.w};
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const int c = 8 * q8 + i;
                float y = fmaf(__uint_as_float(x[c]), p.scale, -mm[i]);
                if (masked) y = (vis[c >> 5] >> (c & 31)) & 1u ? y : -INFINITY;
                top = fmaxf(top, y);
                x[c] = __float_as_uint(y);
              }
            }
          }
        };
        shift();
        if (vote_any<128>(1 + wg, top > kRaise)) {
          // New maxima of the columns that need one, from the scores themselves.
          load_scores();
#pragma unroll
          for (int g = 0; g < G32; ++g) {
            if (32 * g < live) {
              float y[32];
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                y[i] = __uint_as_float(x[32 * g + i]) * p.scale;
                if (masked) y[i] = (vis[g] >> i) & 1u ? y[i] : -INFINITY;
              }
              red[quad * N + 32 * g + lane] = transpose_reduce(y, lane, [](float a, float b) { return fmaxf(a, b); });
            }
          }
          named_bar_sync(1 + wg, 128);
          if (wg_tid < live) {
            const float t = fmaxf(fmaxf(red[wg_tid], red[N + wg_tid]), fmaxf(red[2 * N + wg_tid], red[3 * N + wg_tid]));
            const float old = m_ref[wg_tid];
            const bool raise = old == kUnset ? t > kUnset : t > old + kRaise;
            factor[wg_tid] = raise ? (old == kUnset ? 0.f : exp2f(old - t)) : 1.f;
            if (raise) m_ref[wg_tid] = t;
          }
          named_bar_sync(1 + wg, 128);
          if (kt > s.k0) {
            // O of the tiles before this one is complete once the product of tile j - 1 is.
            wait(done + 8 * ((j - 1) & 1), ((j - 1) >> 1) & 1);
            tc_fence_after();
#pragma unroll
            for (int g = 0; g < G32; ++g) {
              if (32 * g < live) {
                uint32_t o[32];
                const uint32_t addr = lanes + 2 * N + (seg & 1) * N + c0 + 32 * g;
                tmem_ld32_nowait(addr, o);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                  const float f = 32 * g + i < live ? factor[32 * g + i] : 1.f;
                  o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                  l[32 * g + i] *= f;
                }
                tmem_store32(addr, o);
              }
            }
          }
          load_scores();
          shift();
        }
        if (masked) {
          // Rows of V without a key are whatever lay there: cleared. A drafted value that is not finite would reach
          // every column as 0 * inf: it is cleared too, and added at the end to the columns that see it.
          const int node = key - s.r.pad;
          const bool in_prefix = key < s.r.len, in_tree = node >= 0 && node < s.r.n;
          wait(v_full + 8 * stage, (j / S::kStages) & 1);
          if (wg < S::kHalves) {
            const uint32_t row = sV(stage) + wg * kHalf + r * 128;
            if (!in_prefix && !in_tree) {
#pragma unroll
              for (int c = 0; c < 8; ++c)
                asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(row + 16 * (c ^ (r & 7))), "r"(0) : "memory");
            } else if (in_tree) {
              constexpr uint32_t e = DT == AF_DTYPE_BF16 ? 0x7f80u : 0x7c00u;
#pragma unroll
              for (int c = 0; c < 8; ++c) {
                const uint32_t where = row + 16 * (c ^ (r & 7));
                uint32_t w[4];
                asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(where) : "memory");
                bool bad = false;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const bool lo = (w[i] & e) == e, hi = ((w[i] >> 16) & e) == e;
                  w[i] &= (lo ? 0u : 0xffffu) | (hi ? 0u : 0xffff0000u);
                  bad |= lo || hi;
                }
                if (bad) {
                  sick = true;
                  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(where), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
                }
              }
            }
          }
        }
        // P^T row of this key: 16-byte pieces of 8 columns.
        const uint32_t prow = sK(stage) + (N == 128 ? wg * kHalf : 0) + r * 128;
#pragma unroll
        for (int q8 = 0; q8 < C / 8; ++q8) {
          if (8 * q8 < live) {
            float e[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              e[i] = ex2(__uint_as_float(x[8 * q8 + i]));
              l[8 * q8 + i] += e[i];
            }
            const int piece = (N == 128 ? 0 : 4 * wg) + q8;
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(prow + 16 * (piece ^ (r & 7))), "r"(pack2<DT>(e[0], e[1])),
                         "r"(pack2<DT>(e[2], e[3])), "r"(pack2<DT>(e[4], e[5])), "r"(pack2<DT>(e[6], e[7]))
                         : "memory");
          }
        }
        fence_proxy_async_smem();  // P (and V) are read by the tensor cores
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full + 8 * sb);
      }
      // ---- the segment's rows: O^T lane = dim, column = row ----
      named_bar_sync(1 + wg, 128);  // the last factors are read
#pragma unroll
      for (int g = 0; g < G32; ++g)
        if (32 * g < live) red[quad * N + 32 * g + lane] = transpose_reduce(l + 32 * g, lane, [](float a, float b) { return a + b; });
      wait(o_full + 8 * (seg & 1), (seg >> 1) & 1);
      tc_fence_after();
      named_bar_sync(1 + wg, 128);
      if (wg_tid < live) factor[wg_tid] = (red[wg_tid] + red[N + wg_tid]) + (red[2 * N + wg_tid] + red[3 * N + wg_tid]);
      const bool set_aside = vote_any<256>(3, sick);  // (and the sums are there)
      const bool whole = s.whole();
      const int which = s.k0 == 0 ? 1 : 0;
      float* part = scratch.sums(blockIdx.x, which) + (int64_t)c0 * HD;
      int node = c0 / p.group, head = c0 % p.group;
      const int64_t first = s.r.s0 + (int64_t)s.qt * p.nt;
      // The values of dim r that are not finite among the segment's nodes that node i sees.
      auto aside = [&](int i) {
        float sum = 0.f;
        for (int x = max(0, s.k0 * kKeys - s.r.pad); x < min(s.r.n, s.k1 * kKeys - s.r.pad); ++x) {
          const float y = load_scalar<DT>(p.v_rows + (int64_t)(s.r.s0 + x) * p.v_n + s.kvh * p.v_h, r);
          if (!isfinite(y) && (seen_bits(p, s, i, x) & 1u)) sum += y;
        }
        return sum;
      };
#pragma unroll
      for (int g = 0; g < G32; ++g) {
        if (32 * g < live) {
          uint32_t o[32];
          tmem_ld32_nowait(lanes + 2 * N + (seg & 1) * N + c0 + 32 * g, o);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const int c = 32 * g + i;
            if (c < live && r < HD) {
              float y = __uint_as_float(o[i]);
              if (set_aside) y += aside(s.qt * p.nt + node);
              if (whole) {
                const float sum = factor[c];
                y = sum == 0.f ? 0.f : y / sum;
                *reinterpret_cast<uint16_t*>(p.out + (first + node) * p.out_n + (s.kvh * p.group + head) * p.out_h + 2 * r) = to_bits<DT>(y);
              } else {
                part[(int64_t)c * HD + r] = y;
              }
              if (++head == p.group) {
                head = 0;
                ++node;
              }
            }
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(o_empty + 8 * (seg & 1));
      if (wg_tid < live) {
        const float m = m_ref[wg_tid], sum = factor[wg_tid];
        if (!whole) {
          scratch.stats(blockIdx.x, which)[c0 + wg_tid] = make_float2(m, sum);
        } else if (p.lse) {
          const int c = c0 + wg_tid;
          p.lse[(first + c / p.group) * p.heads + s.kvh * p.group + c % p.group] =
              sum == 0.f ? -INFINITY : (m + log2f(sum)) * 0.6931471805599453f;
        }
      }
      if (!whole && s.k0 == 0) {
        wrote_start = true;
        if (tid == 0) {
          const int64_t last = (s.row_end * ctas - 1) / all;  // the CTA with the row's last tile
          *scratch.started(blockIdx.x) = Started{(int)last, (int)first, cols, s.kvh};
        }
      }
      ++seg;
    }
    if (!wrote_start && tid == 0) scratch.started(blockIdx.x)->last = 0;
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && *failed && p.status) atomicOr(p.status, AF_STATUS_TIMEOUT);
  if (warp == kSoft) {
    tc_fence_after();
    tmem_dealloc(tmem, 4 * N);
  }
}

constexpr int kJoinThreads = 256;
constexpr int kJoinBlocks = 16;  // per CTA of the main kernel

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
  for (int row = share ? blockIdx.y : blockIdx.y * W + warp; row < st.rows; row += share ? kJoinBlocks : kJoinBlocks * W) {
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

int64_t workspace_bytes() { return Scratch<128, 128>::bytes(sm_count()); }

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
  const cudaError_t attr = cudaFuncSetAttribute(k_tree_attention<DT, N, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes);
  if (attr != cudaSuccess) return fail(AF_ERR_CUDA, std::string("af_tree_attention: ") + cudaGetErrorString(attr));
  const int ctas = sm_count();
  cudaError_t e = launch_ex(k_tree_attention<DT, N, HD>, dim3(ctas), dim3(kThreads), (size_t)S::kBytes, s, false, dim3(1), p);
  if (e == cudaSuccess && p.capacity + p.total > kKeys)  // else every row is one tile
    e = launch_ex(k_tree_attention_join<DT, N, HD>, dim3(ctas, kJoinBlocks), dim3(kJoinThreads), 0, s, true, dim3(1), p, ctas);
  if (e != cudaSuccess) return fail(AF_ERR_CUDA, std::string("af_tree_attention: launch: ") + cudaGetErrorString(e));
  return check_launch("af_tree_attention");
}

template <int DT>
int launch_shape(const Params& p, int n, int64_t head_dim, cudaStream_t s) {
  if (head_dim == 128) return n == 64 ? launch<DT, 64, 128>(p, s) : launch<DT, 128, 128>(p, s);
  return n == 64 ? launch<DT, 64, 64>(p, s) : launch<DT, 128, 64>(p, s);
}

}  // namespace
}  // namespace af

using namespace af;

extern "C" int af_tree_attention_workspace_bytes(int64_t* bytes) {
  AF_REQUIRE(bytes, "af_tree_attention_workspace_bytes: null pointer");
  *bytes = workspace_bytes();
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
  // Columns of a tile: 64 when the average tree fits, else 128 (the keys are read once per row tile).
  const int n = ceil_div(a.total, a.batch) * group <= 64 ? 64 : 128;
  const int box = (int)(a.page_size % 32 == 0 ? 32 : a.page_size % 16 == 0 ? 16 : 8);
  p.nt = n / group;
  const uint64_t hd = (uint64_t)a.head_dim, kvh = (uint64_t)a.n_kv_heads;
  {
    const uint64_t dims[3] = {hd, (uint64_t)a.n_heads, (uint64_t)a.total};
    const int64_t st[2] = {a.q_strides[1], a.q_strides[0]};
    const uint32_t bx[3] = {64, (uint32_t)group, (uint32_t)p.nt};
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
  cudaStream_t s = as_stream(stream);
  return a.dtype == AF_DTYPE_BF16 ? launch_shape<AF_DTYPE_BF16>(p, n, a.head_dim, s) : launch_shape<AF_DTYPE_F16>(p, n, a.head_dim, s);
}
