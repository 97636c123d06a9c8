// Eviction of cached tokens by the attention weight that they were given (sm_100a).
//
// Every (layer, request, head) is a segment of its own. k_select finds, one CTA
// per segment, the smallest weight that stays: a radix selection over the
// weights' bits, 11, 11 and 10 of them at a time, each a histogram of the
// tokens that still tie, and then writes the places that stay in order. k_move
// brings their rows to the front, in place: row r comes from kept[r] >= r,
// and a step stores rows that no later step loads, so between a step's loads
// and its stores lies one barrier and nothing else; the loads of the next two steps
// are in flight meanwhile. Columns of a row are independent: keys and
// values, and with few segments 64 or 128 bytes of them, are CTAs of their own, and
// with fewer still a cluster shares each step's rows.
//
// k_move is bound by HBM: every moved byte is read and written once. k_select is bound by latency: three passes over weights, of
// which a thread holds the first eight in registers, and one in order, with a barrier for each 512 places (122 -> 113 us for the second).
//   One request of 4100 tokens down to 2048, 28 layers of 4 heads x 128 in 4 bits: 36 us; the bytes need 12.
//   16 requests of 900 to 4100 down to 1500, 6 layers of 4 heads x 128 in 16 bits: 113 us; the bytes need 74.
// (Rows one by one instead of a warp's rows together 338 us for the second, a binary search for the threshold instead of
// histograms 11 us more for the first and 25 for the second.)
#include <string>

#include "int4_cache.cuh"
#include "tree.cuh"

namespace af {
namespace kv_evict {
namespace {

struct SelectArgs {
  const int* lengths;
  const float* weights;
  int64_t wl, wr, wh;  // strides: layer, request, head
  int* kept;
  float* weights_out;
  int* lengths_out;
  int batch, heads, places, keep, sinks, recent;
  int64_t capacity;
  unsigned* status;
};

constexpr int kSelThreads = 512, kSelWarps = kSelThreads / 32, kBins = 2048, kOwn = kBins / kSelThreads;
constexpr int kHeld = 8;  // places of a thread whose weights stay in registers

// Ascending whole numbers for ascending weights; -0 equals 0, and NaN is above all numbers.
__device__ __forceinline__ uint32_t order_of(float w) {
  if (isnan(w)) return 0xffffffffu;
  const uint32_t b = __float_as_uint(w + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__global__ void __launch_bounds__(kSelThreads) k_select(const SelectArgs a) {
  __shared__ int s_hist[kBins];
  __shared__ int s_sum[2][kSelWarps];
  __shared__ int s_bin, s_need;
  pdl_trigger();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t seg = blockIdx.x;
  const int h = (int)(seg % a.heads), b = (int)(seg / a.heads % a.batch);
  const int64_t l = seg / a.heads / a.batch;
  const int given = a.lengths[b];
  const bool bad = given < 0 || given > a.capacity || given > a.places;
  const int t = bad ? 0 : given;
  const float* w = a.weights + l * a.wl + b * a.wr + h * a.wh;
  int* kept = a.kept + seg * a.keep;
  float* out = a.weights_out + seg * a.places;
  if (tid == 0 && l == 0 && h == 0) {
    a.lengths_out[b] = bad ? given : min(t, a.keep);
    if (bad && a.status) atomicOr(a.status, AF_STATUS_BOUNDS);
  }
  if (t <= a.keep) {  // all stay
    for (int i = tid; i < a.keep; i += kSelThreads) kept[i] = i < t ? i : -1;
    // (all of them where the length is none: whoever takes the result's weights over loses nothing)
    for (int i = tid; i < a.places; i += kSelThreads) out[i] = i < t || bad ? w[i] : 0.f;
    return;
  }
  // The weights of places [lo, hi) decide; need of them stay (keep >= sinks + recent, t > keep: hi - lo > need).
  const int lo = a.sinks, hi = t - a.recent, need0 = a.keep - a.sinks - a.recent;
  uint32_t held[kHeld];
#pragma unroll
  for (int c = 0; c < kHeld; ++c) held[c] = c * kSelThreads + tid < t ? order_of(w[c * kSelThreads + tid]) : 0;
  // f(place, order of its weight) for the thread's places, and some behind the last token.
  auto for_places = [&](auto f) {
#pragma unroll
    for (int c = 0; c < kHeld; ++c)
      if (c * kSelThreads < t) f(c * kSelThreads + tid, held[c]);
#pragma unroll 4
    for (int i0 = kHeld * kSelThreads; i0 < t; i0 += kSelThreads) f(i0 + tid, i0 + tid < t ? order_of(w[i0 + tid]) : 0u);
  };
  uint32_t prefix = 0;
  int need = need0;
  if (need0 > 0) {
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, above = pass == 0 ? 32 : shift + (pass == 1 ? 11 : 10);
      const uint32_t mask = pass == 2 ? 1023u : 2047u;
#pragma unroll
      for (int i = 0; i < kOwn; ++i) s_hist[tid + i * kSelThreads] = 0;
      __syncthreads();
      for_places([&](int i, uint32_t k) {
        if (i >= lo && i < hi && (pass == 0 || k >> above == prefix >> above)) atomicAdd(&s_hist[(k >> shift) & mask], 1);
      });
      __syncthreads();
      // Thread x has kOwn bins, from 2047 - kOwn x on downwards; from the top down, the one in which the need-th token lies.
      int c[kOwn], upto = 0;
#pragma unroll
      for (int i = 0; i < kOwn; ++i) upto += c[i] = s_hist[kBins - 1 - kOwn * tid - i];
      const int mine = upto;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
      }
      if (lane == 31) s_sum[0][warp] = upto;
      __syncthreads();
      const int before = __reduce_add_sync(0xffffffffu, lane < warp ? s_sum[0][lane] : 0);
      int begin = before + upto - mine;
#pragma unroll
      for (int i = 0; i < kOwn; ++i) {
        if (begin < need && need <= begin + c[i]) {
          s_bin = kBins - 1 - kOwn * tid - i;
          s_need = need - begin;
        }
        begin += c[i];
      }
      __syncthreads();
      prefix |= (uint32_t)s_bin << shift;
      need = s_need;
    }
  }
  // Tokens above `prefix` stay, and the first `need` of those that equal it. In order: the number of certain ones and of equal
  // ones before each, both in one word (a chunk has fewer than 2^16 places).
  int certain = 0, equal = 0, turn = 0;
  for_places([&](int i, uint32_t k) {
    const bool middle = i >= lo && i < hi;
    const bool sure = i < t && (!middle || (need0 > 0 && k > prefix)), tie = middle && need0 > 0 && k == prefix;
    const uint32_t sures = __ballot_sync(0xffffffffu, sure), ties = __ballot_sync(0xffffffffu, tie);
    if (lane == 0) s_sum[turn][warp] = __popc(sures) | __popc(ties) << 16;
    __syncthreads();
    const int all = lane < kSelWarps ? s_sum[turn][lane] : 0;
    const int before = __reduce_add_sync(0xffffffffu, lane < warp ? all : 0), total = __reduce_add_sync(0xffffffffu, all);
    const uint32_t below = (1u << lane) - 1u;
    const int sure_at = certain + (before & 0xffff) + __popc(sures & below), tie_at = equal + (before >> 16) + __popc(ties & below);
    if (sure || (tie && tie_at < need)) {
      const int at = sure_at + min(tie_at, need);
      kept[at] = i;
      out[at] = w[i];
    }
    certain += total & 0xffff;
    equal += total >> 16;
    turn ^= 1;
  });
  for (int i = a.keep + tid; i < a.places; i += kSelThreads) out[i] = 0.f;
}

struct MoveArgs {
  char *k, *v;                                      // 16-bit rows; 4 bits: k alone
  int64_t kl, kp, kt, kh, vl, vp, vt, vh;           // byte strides: layer, page, token (16-bit rows), head
  const int *tables, *lengths, *kept;
  int64_t tables_ld, capacity;
  int batch, heads, pages, page, places, keep;
  int columns, pieces;                              // CTAs side by side of a row; pieces of 16 (of 4 bits and 64 dims: 8) bytes of each
  int rows;                                         // of a warp's step: at most 32, and Move::kPieces pieces
  uint32_t by_pieces;                               // p / pieces = p * by_pieces >> 20 for p < 2048, pieces <= 256
  unsigned* status;
};

constexpr int kMoveThreads = 256, kMoveWarps = kMoveThreads / 32, kStages = 3;  // steps in flight

// Where a row lies: its first piece, and its row of a 4-bit block.
struct Place {
  char* at;
  int r;
};

// HD = 0: rows of 16 bits (or any other) type; 64 or 128: 4-bit blocks of that many dims.
template <int HD>
struct Move {
  static constexpr int kBytes = HD == 64 ? 8 : 16;             // of a piece
  static constexpr int kPieces = HD == 0 ? 256 : 5 * 32;       // of a warp's step
  static constexpr int kData = kStages * kMoveWarps * kPieces * kBytes;
  static constexpr int kPlaces = kMoveWarps * 32 * (int)sizeof(Place);  // of a step's rows: where from, and per stage where to
  static constexpr int kShared = kData + (1 + kStages) * kPlaces;
};

template <int BYTES>
__device__ __forceinline__ void copy_in(uint32_t dst, const char* src) {
  if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}

// CLUSTER CTAs share each step's rows. A warp's step: its lanes look up a row each (page and place, where from and where to), then move the rows' pieces together.
template <int HD, int CLUSTER>
__global__ void __launch_bounds__(kMoveThreads) k_move(const MoveArgs a) {
  using B = kv4::Block<HD == 0 ? 64 : HD>;
  using M = Move<HD>;
  constexpr int kBytes = M::kBytes, kWarpPieces = M::kPieces, kPer = kWarpPieces / 32;
  extern __shared__ __align__(16) uint8_t buf[];
  pdl_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t item = blockIdx.x / CLUSTER;
  const int rank = CLUSTER > 1 ? blockIdx.x % CLUSTER : 0;
  const int column = (int)(item % a.columns);
  const int64_t seg = item / a.columns;
  const int h = (int)(seg % a.heads), b = (int)(seg / a.heads % a.batch);
  const int64_t l = seg / a.heads / a.batch;
  const int t = a.lengths[b];
  if (t <= a.keep || t > a.capacity || t > a.places) return;
  const int* kept = a.kept + seg * a.keep;
  const int* table = a.tables + b * a.tables_ld;
  // Rows before the first gap stay where they are: kept[r] - r never falls.
  int first = 0;
  for (int n = a.keep; n > 0;) {
    const int step = (n + 31) / 32, at = lane * step;
    const int stay = __popc(__ballot_sync(0xffffffffu, at < n && kept[first + min(at, n - 1)] == first + at));
    first += stay ? (stay - 1) * step + 1 : 0;
    n = stay ? min(step - 1, n - (stay - 1) * step - 1) : 0;
  }
  const int step_rows = CLUSTER * kMoveWarps * a.rows;
  const int steps = (a.keep - first + step_rows - 1) / step_rows;
  const int mine = first + (rank * kMoveWarps + warp) * a.rows;  // the warp's first row of step 0
  char* base;
  int64_t page_step, token_step = 0;
  const int half = a.columns / 2;
  if constexpr (HD == 0) {
    const bool val = column >= half;
    base = (val ? a.v + l * a.vl + h * a.vh : a.k + l * a.kl + h * a.kh) + (int64_t)(val ? column - half : column) * a.pieces * 16;
    page_step = val ? a.vp : a.kp;
    token_step = val ? a.vt : a.kt;
  } else {
    base = a.k + l * a.kl + h * a.kh + (int64_t)column * B::kPart;  // columns: keys and values
    page_step = a.kp;
  }
  auto locate = [&](int place) -> Place {
    const int entry = place / a.page, off = place - entry * a.page, pg = table[entry];
    if (pg < 0 || pg >= a.pages) return {nullptr, 0};
    char* at = base + pg * page_step;
    if constexpr (HD == 0) return {at + off * token_step, 0};
    return {at + (int64_t)(off / kv4::kBlockTokens) * B::kBytes, off % kv4::kBlockTokens};
  };
  auto piece_of = [&](const Place& p, int piece) -> char* {
    if constexpr (HD == 0) return p.at + piece * 16;
    return p.at + (piece == 4 ? B::pair(p.r, 0) : B::word(p.r, piece * (kBytes / 4)));
  };
  uint8_t* data = buf + warp * kWarpPieces * kBytes;                     // + stage * kMoveWarps * kWarpPieces * kBytes
  Place* from = reinterpret_cast<Place*>(buf + M::kData) + warp * 32;
  Place* to = from + kMoveWarps * 32;                                    // + stage * kMoveWarps * 32
  bool bad = false;
  auto load = [&](int step) {
    if (step < steps) {
      const int row = mine + step * step_rows + lane;
      __syncwarp();
      if (lane < a.rows) {
        Place src{nullptr, 0}, dst{nullptr, 0};
        if (row < a.keep) {
          src = locate(kept[row]);
          dst = locate(row);
          if (!src.at || !dst.at) bad = true, src.at = nullptr;
        }
        from[lane] = src;
        to[(step % kStages) * kMoveWarps * 32 + lane] = {src.at ? dst.at : nullptr, dst.r};
      }
      __syncwarp();
#pragma unroll
      for (int u = 0; u < kPer; ++u) {
        const int p = lane + 32 * u, row = (int)((uint32_t)p * a.by_pieces >> 20);
        if (row < a.rows) {
          const Place src = from[row];
          if (src.at) copy_in<kBytes>(smem_u32(data) + ((step % kStages) * kMoveWarps * kWarpPieces + p) * kBytes, piece_of(src, p - row * a.pieces));
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll 1
  for (int s = 0; s < kStages - 1; ++s) load(s);
#pragma unroll 1
  for (int s = 0; s < steps; ++s) {
    load(s + kStages - 1);
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
    // All loads of this step have landed: its stores may go over them.
    if constexpr (CLUSTER > 1) cluster_sync_all();
    else __syncthreads();
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      const int p = lane + 32 * u, row = (int)((uint32_t)p * a.by_pieces >> 20);
      if (row < a.rows) {
        const Place dst = to[(s % kStages) * kMoveWarps * 32 + row];
        if (dst.at) {
          char* at = piece_of(dst, p - row * a.pieces);
          const uint8_t* x = data + ((s % kStages) * kMoveWarps * kWarpPieces + p) * kBytes;  // (what this lane itself brought)
          if constexpr (kBytes == 16) *reinterpret_cast<uint4*>(at) = *reinterpret_cast<const uint4*>(x);
          else *reinterpret_cast<uint2*>(at) = *reinterpret_cast<const uint2*>(x);
        }
      }
    }
  }
  if (bad && a.status) atomicOr(a.status, AF_STATUS_BOUNDS);
}

template <int HD, int CLUSTER>
cudaError_t launch_move(const MoveArgs& a, int64_t segments, cudaStream_t s) {
  constexpr int bytes = Move<HD>::kShared;
  // The same for every call: set each time, which costs less than keeping track of the devices.
  const cudaError_t e = cudaFuncSetAttribute(k_move<HD, CLUSTER>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return e;
  return launch_ex(k_move<HD, CLUSTER>, dim3((unsigned)(segments * a.columns * CLUSTER)), dim3(kMoveThreads), (size_t)bytes, s, true, dim3(CLUSTER), a);
}

// Of a CTA of 46 to 112 KB two or four fit an SM. Clusters as long as all of their CTAs do at once. One request of 4100 tokens
// down to 2048, 4 heads x 128 in 4 bits, by clusters of 1, 2, 4 and 8: one layer 28, 23, 19 and 16 us, 14 layers 32, 29, 31 and 35,
// 28 layers 36, 46, 48 and 55. (Clusters that need a second wave, from a replayed graph: 20 layers 47 us with two CTAs, 39 with one.)
template <int HD>
cudaError_t move(const MoveArgs& a, int64_t segments, cudaStream_t s) {
  constexpr int fit = 233472 / (Move<HD>::kShared + 1024);  // of an SM's shared memory
  const int64_t ctas = segments * a.columns, room = fit * sm_count();
  if (8 * ctas <= room) return launch_move<HD, 8>(a, segments, s);
  if (4 * ctas <= room) return launch_move<HD, 4>(a, segments, s);
  return 2 * ctas <= room ? launch_move<HD, 2>(a, segments, s) : launch_move<HD, 1>(a, segments, s);
}

}  // namespace
}  // namespace kv_evict
}  // namespace af

using namespace af;

extern "C" int af_evict_cache(const af_evict_args* args, uint32_t* status, void* stream) {
  AF_REQUIRE(args, "af_evict_cache: null pointer");
  const af_evict_args& w = *args;
  const bool packed = w.int4.head_dim != 0;
  const int64_t layers = packed ? w.int4.layers : w.layers, pages = packed ? w.int4.pages : w.pages, heads = packed ? w.int4.heads : w.heads,
                page = packed ? w.int4.page_size : w.page_size;
  AF_REQUIRE(layers >= 0 && pages >= 0 && heads >= 0 && w.batch >= 0 && w.max_pages >= 0 && w.places >= 0, "af_evict_cache: bad shape");
  AF_REQUIRE(w.sinks >= 0 && w.recent >= 0 && w.keep >= 0 && w.sinks <= w.keep && w.recent <= w.keep - w.sinks,
             "af_evict_cache: sinks and recent must not be negative, and together not more than keep");
  AF_REQUIRE(page > 0 && page <= (1 << 20), "af_evict_cache: bad page_size");
  if (packed) {
    AF_REQUIRE(page % 8 == 0, "af_evict_cache: page_size must be a multiple of 8");
    AF_REQUIRE(w.int4.head_dim == 64 || w.int4.head_dim == 128, "af_evict_cache: head_dim must be 64 or 128");
  } else {
    AF_REQUIRE(w.head_bytes >= 0 && w.head_bytes <= 4096, "af_evict_cache: at most 4096 bytes per head");
  }
  const int64_t segments = layers * w.batch * heads;
  if (w.batch == 0 || layers == 0 || heads == 0) return AF_OK;
  AF_REQUIRE(layers <= (1 << 20) && heads <= (1 << 16) && w.batch <= (1 << 20) && segments <= (1 << 24) && pages <= 0x7fffffff &&
                 w.places <= (1 << 30) && w.keep <= (1 << 30) && w.max_pages <= (1 << 30) && w.max_pages * page <= (1 << 30),
             "af_evict_cache: size too large");
  const bool moves = pages > 0 && w.max_pages > 0 && w.keep > 0 && (packed || w.head_bytes > 0);
  AF_REQUIRE(w.lengths && w.lengths_out && (w.places == 0 || (w.weights && w.weights_out)) && (w.keep == 0 || w.kept), "af_evict_cache: null pointer");
  AF_REQUIRE(!packed || kv4::runs_apart(w.int4, true), "af_evict_cache: the cache's strides let its entries share memory");
  AF_REQUIRE(!moves || (w.tables && (packed ? w.int4.data != nullptr : w.k_cache && w.v_cache)), "af_evict_cache: null pointer");
  kv_evict::SelectArgs a;
  a.lengths = w.lengths;
  a.weights = w.weights;
  a.wl = w.weights_strides[0], a.wr = w.weights_strides[1], a.wh = w.weights_strides[2];
  a.kept = w.kept;
  a.weights_out = w.weights_out;
  a.lengths_out = w.lengths_out;
  a.batch = (int)w.batch;
  a.heads = (int)heads;
  a.places = (int)w.places;
  a.keep = (int)w.keep;
  a.sinks = (int)w.sinks;
  a.recent = (int)w.recent;
  a.capacity = pages ? w.max_pages * page : 0;
  a.status = status;
  kv_evict::MoveArgs m;
  memset(&m, 0, sizeof(m));
  uint64_t al;
  if (packed) {
    m.k = static_cast<char*>(w.int4.data);
    m.kl = w.int4.strides[0], m.kp = w.int4.strides[1], m.kh = w.int4.strides[2];
    al = reinterpret_cast<uintptr_t>(m.k) | (uint64_t)m.kl | (uint64_t)m.kp | (uint64_t)m.kh;
    m.columns = 2;
    m.pieces = 5;
  } else {
    m.k = static_cast<char*>(w.k_cache), m.v = static_cast<char*>(w.v_cache);
    m.kl = w.k_cache_strides[0], m.kp = w.k_cache_strides[1], m.kt = w.k_cache_strides[2], m.kh = w.k_cache_strides[3];
    m.vl = w.v_cache_strides[0], m.vp = w.v_cache_strides[1], m.vt = w.v_cache_strides[2], m.vh = w.v_cache_strides[3];
    al = reinterpret_cast<uintptr_t>(m.k) | reinterpret_cast<uintptr_t>(m.v) | (uint64_t)w.head_bytes;
    for (int i = 0; i < 4; ++i) al |= (uint64_t)w.k_cache_strides[i] | (uint64_t)w.v_cache_strides[i];
    const int whole = (int)(w.head_bytes / 16);
    // Whole rows a CTA where there are many segments for each SM, else 128 or 64 bytes: few long CTAs leave the last ones waiting
    // (384 segments of 256-byte rows: 125 us in 128 bytes, 128 whole).
    m.pieces = 2 * segments < 2 * sm_count() && whole % 4 == 0 ? 4 : 2 * segments < 16 * sm_count() && whole % 8 == 0 ? 8 : whole > 0 ? whole : 1;
    m.columns = whole > 0 ? 2 * (whole / m.pieces) : 2;
  }
  AF_REQUIRE(!moves || (al & 15) == 0, "af_evict_cache: addresses and strides must be multiples of 16 bytes");
  m.by_pieces = (uint32_t)(((1 << 20) + m.pieces - 1) / m.pieces);
  m.rows = packed || 256 / m.pieces > 32 ? 32 : 256 / m.pieces;  // (Move::kPieces)
  m.tables = w.tables;
  m.tables_ld = w.tables_stride;
  m.lengths = w.lengths;
  m.kept = w.kept;
  m.capacity = a.capacity;
  m.batch = a.batch;
  m.heads = a.heads;
  m.pages = (int)pages;
  m.page = (int)page;
  m.places = a.places;
  m.keep = a.keep;
  m.status = status;
  cudaStream_t s = as_stream(stream);
  kv_evict::k_select<<<(unsigned)segments, kv_evict::kSelThreads, 0, s>>>(a);
  if (int st = check_launch("af_evict_cache")) return st;
  if (!moves) return AF_OK;
  const cudaError_t e = !packed ? kv_evict::move<0>(m, segments, s) : w.int4.head_dim == 128 ? kv_evict::move<128>(m, segments, s) : kv_evict::move<64>(m, segments, s);
  if (e != cudaSuccess) return fail(AF_ERR_CUDA, std::string("af_evict_cache: ") + cudaGetErrorString(e));
  return check_launch("af_evict_cache");
}
