// The attention that cached tokens are given, added up (sm_100a).
//
//   weights[b, h, p] += sum over the request's rows i and the query heads of group h of exp(scale q_i . k_p - lse_i)
//
// over the places p that row i sees. The rows' sums are known (lse), so keys
// are independent: a warp takes 32 of them, all rows of the request against
// 16 at a time in registers (m16n8k16, the keys as the M side: few rows waste little), and adds to their
// weights without atomics. The rows of a request and head, 64 at a time, lie in shared memory with their sums. 4-bit
// keys come by bulk copies, a unit ahead of each warp. The bytes are 80 a key and head in 4 bits (256 in 16) and 8
// of its weight; what bounds it is the chain of a warp's unit (operands, products, exponentials), with four warps a scheduler
// (issue 52 %, tensor pipe 28 %, HBM 22 %). See int4_attention.cu for the fragments' order.
//   64 requests of 1 to 4 tokens, 90 to 8000 keys, 28 heads over 4: 50 us in 4 bits; the bytes need 14.
//   The same over keys in 16 bits, which are loaded as they are needed: 65 us; the bytes need 42.
//   One token over 1500 keys: 5.6 us.
// Tried: rows from global memory for each unit (137 us), keys looked up and loaded unit by unit (70); four chains of products
// (53), 16 keys at a time with two or three CTAs an SM (54, 56), shares by rows as well as units (53 to 59): slower.
#include <string>
#include <type_traits>

#include "int4_attention.cuh"

namespace af {
namespace kv4 {
namespace {

// -lse of a row that gives nothing: one behind the last, or whose lse is -inf. It is added as 2^-kNothing = 0, but what
// a key that is not finite makes of that is not: units whose sums are not finite are added up once more without such rows (to leave
// them out at once takes 53 us instead of 51 for the 64 requests).
constexpr float kNothing = -3.402823466e38f;
constexpr int kUnit = 32, kThreads = 256, kCtas = 2, kRows = 64;  // keys of a unit; CTAs per SM; rows in shared memory at once

struct WeightArgs {
  Params p;                     // q, tables, lengths, starts, window, sinks, scale; data: the cache
  int64_t d_token;              // 16-bit keys: byte stride of a token
  const float* lse;             // [total, heads]
  float* weights;
  int64_t w_request, w_head;    // strides in elements
  int64_t places;
};

__device__ __forceinline__ int units_of(const WeightArgs& a, int b, Request<kUnit>& r) {
  r = request<kUnit>(a.p, b);
  r.bad |= r.len > a.places;
  return r.bad || r.n == 0 ? 0 : r.cached * a.p.kv_heads;
}

template <int DT>
__device__ __forceinline__ void mma(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  if constexpr (DT == AF_DTYPE_BF16) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  } else {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}

// Dynamic shared memory: two units' 4-bit keys per warp.
template <int HD>
constexpr int kRing = kThreads / 32 * 2 * (kUnit / kBlockTokens) * Block<HD>::kPart;

template <int DT, int HD, bool INT4>
__global__ void __launch_bounds__(kThreads, kCtas) k_weights(const __grid_constant__ WeightArgs a) {
  using B = Block<HD>;
  constexpr int W = kThreads / 32, KS = HD / 16;
  __shared__ int s_share[4];  // first unit, the one behind the last; the request that the share begins with, and the units before it
  __shared__ __align__(16) uint4 s_q[kRows * (HD / 8)];
  __shared__ float s_sum[kRows];  // -lse in log2 units, or kNothing
  __shared__ int s_first[kRows];  // first place of the row's window
  __shared__ __align__(8) uint64_t s_full[2 * W];
  extern __shared__ __align__(128) uint8_t ring[];
  constexpr int kUnitBytes = kUnit / kBlockTokens * B::kPart;
  const Params& p = a.p;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  Request<kUnit> r;
  if (tid < 2 * W) {
    mbar_init(smem_u32(s_full + tid), 1);
    fence_barrier_init();
  }
  if (warp == 0) {
    bool disorder = false;
    int all = 0;
    for (int b = lane; b < p.batch; b += 32) {
      all += units_of(a, b, r);
      disorder |= p.starts[b + 1] < p.starts[b];
      if (r.bad && blockIdx.x == 0 && p.status) atomicOr(p.status, AF_STATUS_BOUNDS);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
    if (__any_sync(0xffffffffu, disorder)) all = 0;  // rows of several requests: no work
    const int each = all / (int)gridDim.x, more = all - each * (int)gridDim.x, c = blockIdx.x;
    const int first = each * c + min(c, more), end = each * (c + 1) + min(c + 1, more);
    int before = 0, b0 = 0;
    if (first < end) {
      for (;; b0 += 32) {
        int upto = b0 + lane < p.batch ? units_of(a, b0 + lane, r) : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += y;
        }
        const uint32_t behind = __ballot_sync(0xffffffffu, first < before + upto);
        if (behind) {
          const int x = __ffs(behind) - 1;
          b0 += x;
          before += x ? __shfl_sync(0xffffffffu, upto, x - 1) : 0;
          break;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
      }
    }
    if (lane == 0) s_share[0] = first, s_share[1] = end, s_share[2] = b0, s_share[3] = before;
  }
  __syncthreads();
  const int end = s_share[1];
  int b = s_share[2], before = s_share[3], u0 = s_share[0];
  if (u0 >= end) return;
  int of = units_of(a, b, r);
  const int kap = !INT4 ? g : g & 1 ? 4 + ((g >> 1) ^ 1) : g >> 1;
  uint8_t* slots = ring + warp * 2 * kUnitBytes;
  const uint32_t full = smem_u32(s_full + 2 * warp);
  int brought = 0, taken = 0;  // units of this warp
  bool lost = false;           // a wait has run out
#pragma unroll 1
  while (u0 < end) {
#pragma unroll 1
    while (u0 >= before + of) {
      before += of;
      of = units_of(a, ++b, r);
    }
    // The share's units of one request and head: x0 .. x1 - 1.
    const int h = (u0 - before) / r.cached, x0 = (u0 - before) - h * r.cached, x1 = min(r.cached, x0 + end - u0);
    u0 += x1 - x0;
    const int* table = p.tables + (int64_t)b * p.tables_ld;
    const int rows = r.n * p.group, first_all = p.window ? max(0, r.len - max(0, p.window - r.n)) : 0;
    // The warp's units of the segment, eight at a time: lane 4 y + z knows where block z of the y-th of them lies (null: there is no
    // such key, or its page is none: reads as zeros).
    int known = x0 + warp - 8 * W, next = x0 + warp;
    const char* from = nullptr;
    auto bring = [&]() {
      if (next >= x1 || lost) return;
      if (next - known >= 8 * W) {
        known = next;
        const int x = known + W * (lane >> 2), at = kUnit * (x < r.sink_units ? x : x - r.sink_units + r.from) + kBlockTokens * (lane & 3);
        from = nullptr;
        if (x < x1 && at < r.len) {
          const int entry = entry_of(p, at), page = table[entry];
          if (page >= 0 && page < p.pages)
            from = p.data + page * p.d_page + h * p.d_head + (int64_t)((at - entry * p.page) / kBlockTokens) * B::kBytes;
          else if (p.status)
            atomicOr(p.status, AF_STATUS_BOUNDS);
        }
      }
      const int slot = brought & 1;
      const bool mine = (lane >> 2) * W == next - known;
      uint8_t* to = slots + slot * kUnitBytes + (lane & 3) * B::kPart;
      if (mine && !from) {
        for (int y = 0; y < B::kPart / 16; ++y) reinterpret_cast<uint4*>(to)[y] = make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();
      }
      const uint32_t blocks = __ballot_sync(0xffffffffu, mine && from);
      if (lane == 0) mbar_arrive_expect_tx(full + 8 * slot, __popc(blocks) * B::kPart);
      __syncwarp();
      if (mine && from)
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(to)), "l"(from), "r"(B::kPart),
                     "r"(full + 8 * slot)
                     : "memory");
      ++brought;
      next += W;
    };
#pragma unroll 1
    for (int row0 = 0; row0 < rows; row0 += kRows) {
      if (INT4 && row0 > 0) known = x0 + warp - 8 * W, next = x0 + warp;
      if constexpr (INT4) bring();  // (on its way while the rows are laid out)
      // A row's 16-byte pieces in the order in which the lanes of a quad take them, exchanged by halves of 128 bytes in odd rows:
      // eight lanes read different banks.
      const int count = min(kRows, rows - row0), tiles = (count + 7) / 8;
      __syncthreads();
      for (int i = tid; i < tiles * 8 * (HD / 8); i += kThreads) {
        const int row = i / (HD / 8), c = i % (HD / 8), flat = row0 + row;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (row < count)
          v = *reinterpret_cast<const uint4*>(p.q + (int64_t)(r.s0 + flat / p.group) * p.q_n + (h * p.group + flat % p.group) * p.q_h + 16 * c);
        s_q[row * (HD / 8) + ((c % (KS / 2) * 4 + c / (KS / 2)) ^ (4 * (row & 1)))] = v;
      }
      if (tid < tiles * 8) {
        const int flat = row0 + tid, node = flat / p.group;
        const float lse = tid < count ? a.lse[(int64_t)(r.s0 + node) * p.heads + h * p.group + flat % p.group] : -INFINITY;
        s_sum[tid] = lse == -INFINITY ? kNothing : lse * -1.4426950408889634f;
        s_first[tid] = p.window ? max(0, r.len - max(0, p.window - (node + 1))) : 0;
      }
      __syncthreads();
#pragma unroll 1
      for (int x = x0 + warp; x < x1 && !lost; x += W) {
        if constexpr (INT4) {
          bring();
          // (no attempts, no wait: the copy counts as lost)
          if (p.patience == 0 || !mbar_try_wait(full + 8 * (taken & 1), (taken >> 1) & 1)) {
            int left = p.patience;
            do lost = --left < 0;
            while (!lost && !mbar_try_wait(full + 8 * (taken & 1), (taken >> 1) & 1));
          }
          lost = __any_sync(0xffffffffu, lost);
          if (lost) {
            if (lane == 0 && p.status) atomicOr(p.status, AF_STATUS_TIMEOUT);
            break;
          }
        }
        const int place = kUnit * (x < r.sink_units ? x : x - r.sink_units + r.from);
        // The lane adds up the weight of one key: row kap of block t.
        const int mine = place + 8 * t + kap;
        float* at_weight = a.weights + b * a.w_request + h * a.w_head + mine;
        const float old = mine < r.len ? *at_weight : 0.f;
        const bool masked = place + kUnit > r.len || (p.window && place < first_all && place + kUnit > p.sinks);
        uint32_t k[2][KS][4];  // the operand, 16 keys each: keys kap of two blocks, the 32 (16) dims that the lane takes
        bool bad = false;
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            if constexpr (INT4) {
              const uint8_t* block = slots + (taken & 1) * kUnitBytes + (2 * half + y) * B::kPart;
              uint32_t w[HD / 32];
              if constexpr (HD == 128) {
                const uint4 v = *reinterpret_cast<const uint4*>(block + B::word(kap, 4 * t));
                w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
              } else {
                const uint2 v = *reinterpret_cast<const uint2*>(block + B::word(kap, 2 * t));
                w[0] = v.x, w[1] = v.y;
              }
              const uint32_t pr = *reinterpret_cast<const uint32_t*>(block + B::pair(kap, (HD / 4) * t / kGroup));
              const uint32_t s2 = __byte_perm(pr, 0, 0x1010), o2 = __byte_perm(pr, 0, 0x3232);
#pragma unroll
              for (int i = 0; i < HD / 32; ++i) {
                k[half][2 * i][y] = two_values<DT, 0>(w[i], s2, o2);
                k[half][2 * i][2 + y] = two_values<DT, 1>(w[i], s2, o2);
                k[half][2 * i + 1][y] = two_values<DT, 2>(w[i], s2, o2);
                k[half][2 * i + 1][2 + y] = two_values<DT, 3>(w[i], s2, o2);
              }
            } else {
              const int at = place + 16 * half + 8 * y, entry = entry_of(p, at), page = at < r.len ? table[entry] : 0;
              bad |= page < 0 || page >= p.pages;
              const bool row = page >= 0 && page < p.pages && at + kap < r.len;
              const char* from = p.data + (row ? page : 0) * p.d_page + h * p.d_head + (int64_t)(at - entry * p.page + kap) * a.d_token + t * (HD / 2);
#pragma unroll
              for (int i = 0; i < KS / 2; ++i) {
                const uint4 v = row ? *reinterpret_cast<const uint4*>(from + 16 * i) : make_uint4(0, 0, 0, 0);
                k[half][2 * i][y] = v.x, k[half][2 * i][2 + y] = v.y, k[half][2 * i + 1][y] = v.z, k[half][2 * i + 1][2 + y] = v.w;
              }
            }
          }
        if (bad && p.status) atomicOr(p.status, AF_STATUS_BOUNDS);
        float sum[2][2];  // [half][block]
        const uint4* q_even = s_q + g * (HD / 8) + t + 4 * (g & 1);  // pieces 4 i + t, those of odd rows exchanged
        const uint4* q_odd = s_q + g * (HD / 8) + t + 4 - 4 * (g & 1);
        // careful: row by row, which rows see a key, and which give anything.
        auto add_up = [&](auto careful) {
          sum[0][0] = sum[0][1] = sum[1][0] = sum[1][1] = 0.f;
#pragma unroll 1
          for (int tile = 0; tile < tiles; ++tile) {
            float c[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
            for (int i = 0; i < KS / 2; ++i) {
              const uint4 v = (i & 1 ? q_odd : q_even)[tile * HD + 4 * (i & 2)];
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                mma<DT>(c[half], k[half][2 * i], v.x, v.y);
                mma<DT>(c[half], k[half][2 * i + 1], v.z, v.w);
              }
            }
            const float2 less = *reinterpret_cast<const float2*>(s_sum + 8 * tile + 2 * t);
            if constexpr (decltype(careful)::value) {
              const int2 first = *reinterpret_cast<const int2*>(s_first + 8 * tile + 2 * t);
#pragma unroll
              for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                  const int at = place + 16 * half + 8 * y + kap;
                  const bool in = at < r.len, sink = at < p.sinks;
                  if (in && less.x != kNothing && (sink || at >= first.x)) sum[half][y] += ex2(fmaf(c[half][2 * y], p.scale, less.x));
                  if (in && less.y != kNothing && (sink || at >= first.y)) sum[half][y] += ex2(fmaf(c[half][2 * y + 1], p.scale, less.y));
                }
            } else {
#pragma unroll
              for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int y = 0; y < 2; ++y)
                  sum[half][y] += ex2(fmaf(c[half][2 * y], p.scale, less.x)) + ex2(fmaf(c[half][2 * y + 1], p.scale, less.y));
            }
          }
        };
        bool again = masked;
        if (!masked) {
          add_up(std::false_type{});
          again = !__all_sync(0xffffffffu, sum[0][0] + sum[0][1] + sum[1][0] + sum[1][1] < INFINITY);
        }
        if (again) add_up(std::true_type{});
        float given = 0.f;
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          float x = sum[y >> 1][y & 1];
          x += __shfl_xor_sync(0xffffffffu, x, 1);
          x += __shfl_xor_sync(0xffffffffu, x, 2);
          if (t == y) given = x;
        }
        if (mine < r.len) *at_weight = old + given;
        ++taken;
        __syncwarp();
      }
    }
  }
  // Copies in flight (there is one only when a wait ran out) land before the CTA's shared memory is given up (bounded).
  for (; INT4 && taken < brought; ++taken)
    for (int tries = 0; tries < kPatience && !mbar_try_wait(full + 8 * (taken & 1), (taken >> 1) & 1); ++tries) {
    }
}

template <int DT, int HD>
int launch(const WeightArgs& a, bool int4, cudaStream_t s) {
  const int ctas = sm_count() * kCtas;
  if (int4) {
    if (int st = allow_smem<k_weights<DT, HD, true>>(kRing<HD>, "af_attention_weights")) return st;
    k_weights<DT, HD, true><<<ctas, kThreads, kRing<HD>, s>>>(a);
  } else {
    k_weights<DT, HD, false><<<ctas, kThreads, 0, s>>>(a);
  }
  return check_launch("af_attention_weights");
}

}  // namespace
}  // namespace kv4
}  // namespace af

using namespace af;

extern "C" int af_attention_weights(const af_attention_weights_args* args, uint32_t* status, void* stream) {
  AF_REQUIRE(args, "af_attention_weights: null pointer");
  const af_attention_weights_args& w = *args;
  const af_int4_cache& c = w.cache;
  AF_REQUIRE(w.batch >= 0 && w.total >= 0 && w.max_pages >= 0 && w.places >= 0 && c.pages >= 0, "af_attention_weights: bad shape");
  AF_REQUIRE(w.n_heads > 0 && c.heads > 0 && w.n_heads % c.heads == 0, "af_attention_weights: n_heads must be a multiple of the cache's heads");
  AF_REQUIRE(c.head_dim == 64 || c.head_dim == 128, "af_attention_weights: head_dim must be 64 or 128");
  AF_REQUIRE(c.dtype == AF_DTYPE_F16 || c.dtype == AF_DTYPE_BF16, "af_attention_weights: dtype must be fp16 or bf16");
  AF_REQUIRE(c.page_size > 0 && c.page_size % kv4::kBlockTokens == 0 && c.page_size <= (1 << 20), "af_attention_weights: page_size must be a multiple of 8");
  AF_REQUIRE(w.window >= 0 && w.sinks >= 0 && w.window <= (1 << 30) && w.sinks <= (1 << 30), "af_attention_weights: window and sinks must not be negative");
  AF_REQUIRE(w.total <= (1 << 28) && c.pages <= 0x7fffffff && w.n_heads <= (1 << 16) && w.max_pages <= (1 << 30) && w.max_pages * c.page_size <= (1 << 30) &&
                 w.total * (w.n_heads / c.heads) <= (1 << 30) && w.batch <= (1 << 20),
             "af_attention_weights: size too large");
  // Without pages there is nothing to add, but lengths that say otherwise are reported.
  const bool none = w.max_pages == 0 || c.pages == 0;
  if (w.batch == 0 || w.total == 0 || (none && !status)) return AF_OK;
  AF_REQUIRE(w.q && (none || (c.data && w.tables)) && w.lengths && w.starts && w.lse && (w.places == 0 || w.weights), "af_attention_weights: null pointer");
  AF_REQUIRE((double)c.heads * w.batch * (w.max_pages * c.page_size / kv4::kUnit + 2) < 2147483000.0, "af_attention_weights: more than 2^31 units of 32 keys");
  AF_REQUIRE(w.token_stride > 0 || (w.token_stride == 0 && kv4::runs_apart(c, false)),
             "af_attention_weights: token_stride must be 0 (blocks of 4 bits, whose page and head strides let no entries share memory) or positive");
  uint64_t al = reinterpret_cast<uintptr_t>(w.q) | reinterpret_cast<uintptr_t>(c.data) | (uint64_t)w.q_strides[0] | (uint64_t)w.q_strides[1] |
                (uint64_t)c.strides[1] | (uint64_t)c.strides[2] | (uint64_t)w.token_stride;
  AF_REQUIRE((al & 15) == 0, "af_attention_weights: addresses and strides must be multiples of 16 bytes");
  kv4::WeightArgs a;
  memset(&a, 0, sizeof(a));
  kv4::Params& p = a.p;
  p.q = static_cast<const char*>(w.q), p.q_n = w.q_strides[0], p.q_h = w.q_strides[1];
  p.data = static_cast<const char*>(c.data), p.d_page = c.strides[1], p.d_head = c.strides[2];
  p.tables = w.tables;
  p.tables_ld = w.tables_stride;
  p.lengths = w.lengths;
  p.starts = w.starts;
  p.batch = (int)w.batch;
  p.total = (int)w.total;
  p.heads = (int)w.n_heads;
  p.kv_heads = (int)c.heads;
  p.group = (int)(w.n_heads / c.heads);
  p.pages = (int)c.pages;
  kv4::set_page(p, c.page_size);
  p.capacity = none ? 0 : w.max_pages * c.page_size;
  p.window = (int)w.window;
  p.sinks = (int)w.sinks;
  p.reach = p.window - 1;
  p.scale = (float)(w.scale * 1.4426950408889634);
  p.rows = 8;
  p.status = status;
  p.patience = attention_patience();
  a.d_token = w.token_stride;
  a.lse = w.lse;
  a.weights = w.weights;
  a.w_request = w.weights_strides[0], a.w_head = w.weights_strides[1];
  a.places = w.places;
  cudaStream_t s = as_stream(stream);
  const bool int4 = w.token_stride == 0;
  if (c.dtype == AF_DTYPE_BF16) return c.head_dim == 128 ? kv4::launch<AF_DTYPE_BF16, 128>(a, int4, s) : kv4::launch<AF_DTYPE_BF16, 64>(a, int4, s);
  return c.head_dim == 128 ? kv4::launch<AF_DTYPE_F16, 128>(a, int4, s) : kv4::launch<AF_DTYPE_F16, 64>(a, int4, s);
}
