// Rows into and out of the 4-bit paged cache (sm_100a).
//
// Both kernels are bound by HBM: per token and head of 128 dims 512 bytes of
// 16-bit rows against 160 of the cache. A lane takes 8 dims (16 bytes) of a row, a
// code word; the four lanes of a group of 32 dims share its extremes by two exchanges.
#include <string>

#include "int4_cache.cuh"
#include "tree.cuh"

namespace af {
namespace kv4 {
namespace {

constexpr int kThreads = 256;

struct RowArgs {
  const char *k, *v;  // 16-bit rows: read by the write kernel
  char *k_out, *v_out;
  int64_t kl, kn, kh, vl, vn, vh;  // byte strides of the rows: layer, row, head
  char* data;
  int64_t dl, dp, dh;  // of the cache: layer, page, head
  const int64_t* slots;
  const int* rows;
  int64_t n_rows, count, n_slots;
  int layers, page, heads;
  unsigned* status;
};

template <int DT>
__device__ __forceinline__ float from16(uint32_t bits) {
  if constexpr (DT == AF_DTYPE_BF16) {
    return __uint_as_float(bits << 16);
  } else {
    const __half h = __ushort_as_half((unsigned short)bits);
    return __half2float(h);
  }
}
template <int DT>
__device__ __forceinline__ uint32_t to16(float x) {
  if constexpr (DT == AF_DTYPE_BF16) {
    return f2bf_bits(x);
  } else {
    return __half_as_ushort(__float2half_rn(x));
  }
}
template <int DT>
__device__ __forceinline__ bool finite16(uint32_t bits) {
  constexpr uint32_t e = DT == AF_DTYPE_BF16 ? 0x7f80u : 0x7c00u;
  return (bits & e) != e;
}

// The code of x: (x - offset) / scale rounded half to even, in 0 .. 15, as exact arithmetic rounds it. d = x - offset in
// fp32, scale > 0.
__device__ __noinline__ uint32_t careful_code(float x, float offset, float d, float scale) {
  const float k = fminf(floorf(d / scale), 15.f);
  const float r = fmaf(-(k + 0.5f), scale, d);  // its sign is exact
  // What the difference lost when it was rounded to fp32 decides a tie.
  const float b = d - x, lost = (x - (d - b)) + (-offset - b);
  const bool up = r > 0.f || (r == 0.f && (lost > 0.f || (lost == 0.f && ((int)k & 1))));
  return (uint32_t)fminf(k + (up ? 1.f : 0.f), 15.f);
}

// One lane's code word of 8 values, and its group's pair (the same in the group's four lanes).
template <int DT>
__device__ __forceinline__ void encode(const uint4& x, uint32_t& word, uint32_t& pair) {
  using P = Pair16<DT>;
  auto lo2 = __hmin2_nan(__hmin2_nan(P::make(x.x), P::make(x.y)), __hmin2_nan(P::make(x.z), P::make(x.w)));
  auto hi2 = __hmax2_nan(__hmax2_nan(P::make(x.x), P::make(x.y)), __hmax2_nan(P::make(x.z), P::make(x.w)));
#pragma unroll
  for (int o = 1; o <= 2; o <<= 1) {
    lo2 = __hmin2_nan(lo2, P::make(__shfl_xor_sync(0xffffffffu, bits_of(lo2), o)));
    hi2 = __hmax2_nan(hi2, P::make(__shfl_xor_sync(0xffffffffu, bits_of(hi2), o)));
  }
  const float l0 = from16<DT>(bits_of(lo2) & 0xffffu), l1 = from16<DT>(bits_of(lo2) >> 16);
  const float h0 = from16<DT>(bits_of(hi2) & 0xffffu), h1 = from16<DT>(bits_of(hi2) >> 16);
  const float low = fminf(l0, l1), range = fmaxf(h0, h1) - low;
  const bool sound = !(isnan(l0) || isnan(l1)) && fabsf(range) <= 3.402823466e38f;
  if (!sound) {  // the group stands for NaN
    word = 0;
    pair = (DT == AF_DTYPE_BF16 ? 0x7fc0u : 0x7e00u) << 16;
    return;
  }
  uint32_t s16 = to16<DT>(range / 15.f);
  if (!finite16<DT>(to16<DT>(fmaf(15.f, from16<DT>(s16), low)))) --s16;
  pair = s16 | to16<DT>(low) << 16;
  const float scale = from16<DT>(s16);
  word = 0;
  if (scale == 0.f) return;
  constexpr float magic = 12582912.f;  // 1.5 * 2^23: a number below 2^22 added to it is rounded to a whole one
  // (Where the reciprocal overflows every code takes the careful way.)
  const float inv = scale < 1e-37f ? 0.f : 1.f / scale, half = 0.5f * scale;
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float y = from16<DT>(h ? w[i] >> 16 : w[i] & 0xffffu), d = y - low;
      const float t = fminf(fmaf(d, inv, magic), magic + 15.f);
      // Next to a border between two codes, or past the last: |d - code * scale| is no less than half a step.
      uint32_t c = __float_as_uint(t) & 15u;
      if (fabsf(fmaf(-(t - magic), scale, d)) >= half) c = careful_code(y, low, d, scale);
      word |= c << (4 * i + 16 * h);
    }
  }
}

// A warp takes 32 U code words (keys, then values, of one head after the other) of one row.
template <int DT, int HD, int U, bool WRITE>
__global__ void __launch_bounds__(kThreads) k_rows(const RowArgs a, int chunks) {
  using B = Block<HD>;
  constexpr int W = HD / 8;  // words of a row
  const int lane = threadIdx.x & 31;
  const int item = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);  // (row, chunk)
  const int m = item / chunks, chunk = item - m * chunks, l = blockIdx.y;
  if (m >= a.count) return;
  int64_t slot = a.slots[m];
  int64_t row = WRITE && a.rows ? a.rows[m] : m;
  if (WRITE && (slot < 0 || row < 0)) return;
  if (slot >= a.n_slots || (WRITE && row >= a.n_rows)) {
    if (lane == 0 && a.status) atomicOr(a.status, AF_STATUS_BOUNDS);
    if (WRITE) return;
    slot = -1;
  }
  const int64_t pg = slot < 0x7fffffff ? (int)slot / a.page : slot / a.page;
  const int t = (int)(slot - pg * a.page), r = t % kBlockTokens;
  char* block = a.data + l * a.dl + pg * a.dp + (int64_t)(t / kBlockTokens) * B::kBytes;
  const int words = 2 * W * a.heads, x0 = chunk * 32 * U + lane;
  if constexpr (WRITE) {
    const char* k = a.k + l * a.kl + row * a.kn;
    const char* v = a.v + l * a.vl + row * a.vn;
    uint4 buf[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int x = x0 + 32 * u, h = x / (2 * W), val = x / W % 2, w = x % W;
      buf[u] = x < words ? *reinterpret_cast<const uint4*>((val ? v + h * a.vh : k + h * a.kh) + 16 * w) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int x = x0 + 32 * u, h = x / (2 * W), val = x / W % 2, w = x % W;
      uint32_t word, pair;
      encode<DT>(buf[u], word, pair);
      if (x < words) {
        char* part = block + h * a.dh + val * B::kPart;
        *reinterpret_cast<uint32_t*>(part + B::word(r, w)) = word;
        if (w % 4 == 0) *reinterpret_cast<uint32_t*>(part + B::pair(r, w / 4)) = pair;
      }
    }
  } else {
    char* k = a.k_out + l * a.kl + m * a.kn;
    char* v = a.v_out + l * a.vl + m * a.vn;
    uint32_t word[U], pair[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int x = x0 + 32 * u, h = x / (2 * W), val = x / W % 2, w = x % W;
      const bool there = slot >= 0 && x < words;
      const char* part = block + h * a.dh + val * B::kPart;
      word[u] = there ? *reinterpret_cast<const uint32_t*>(part + B::word(r, w)) : 0;
      pair[u] = there ? *reinterpret_cast<const uint32_t*>(part + B::pair(r, w / 4)) : 0;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int x = x0 + 32 * u, h = x / (2 * W), val = x / W % 2, w = x % W;
      if (x >= words) continue;
      // Word and pair are 0 where there is no slot, and so are the values.
      const uint32_t s2 = __byte_perm(pair[u], 0, 0x1010), o2 = __byte_perm(pair[u], 0, 0x3232);
      const uint4 y = make_uint4(two_values<DT, 0>(word[u], s2, o2), two_values<DT, 1>(word[u], s2, o2), two_values<DT, 2>(word[u], s2, o2),
                                 two_values<DT, 3>(word[u], s2, o2));
      *reinterpret_cast<uint4*>((val ? v + h * a.vh : k + h * a.kh) + 16 * w) = y;
    }
  }
}

template <int DT, int HD, bool WRITE>
void launch(const RowArgs& a, cudaStream_t s) {
  // Four words of a lane in flight where a row has them: rows of 4 heads x 128 dims fill a warp's 128.
  const int words = HD / 4 * a.heads;
  const int u = words > 64 ? 4 : words > 32 ? 2 : 1;
  const int chunks = (int)ceil_div(words, 32 * u);
  const dim3 grid((unsigned)ceil_div((int64_t)chunks * a.count, kThreads / 32), (unsigned)a.layers);
  if (u == 4) k_rows<DT, HD, 4, WRITE><<<grid, kThreads, 0, s>>>(a, chunks);
  else if (u == 2) k_rows<DT, HD, 2, WRITE><<<grid, kThreads, 0, s>>>(a, chunks);
  else k_rows<DT, HD, 1, WRITE><<<grid, kThreads, 0, s>>>(a, chunks);
}

template <bool WRITE>
int rows_call(const af_int4_rows* w, uint32_t* status, void* stream, const char* name) {
  const std::string what = std::string(name) + ": ";
  AF_REQUIRE(w, what + "null pointer");
  const af_int4_cache& c = w->cache;
  AF_REQUIRE(c.layers >= 0 && c.pages >= 0 && c.heads >= 0 && w->count >= 0 && w->n_rows >= 0, what + "bad shape");
  AF_REQUIRE(c.page_size > 0 && c.page_size % kBlockTokens == 0, what + "page_size must be a positive multiple of 8");
  AF_REQUIRE(c.head_dim == 64 || c.head_dim == 128, what + "head_dim must be 64 or 128");
  AF_REQUIRE(c.dtype == AF_DTYPE_F16 || c.dtype == AF_DTYPE_BF16, what + "dtype must be fp16 or bf16");
  if (c.layers == 0 || c.heads == 0 || w->count == 0) return AF_OK;
  AF_REQUIRE(w->slots && ((WRITE && w->n_rows == 0) || (w->k && w->v)) && (c.pages == 0 || c.data), what + "null pointer");
  AF_REQUIRE(c.heads <= (1 << 16) && c.page_size <= (1 << 20) && c.layers <= 65535 && c.pages <= 0x7fffffff, what + "size too large");
  uint64_t al = reinterpret_cast<uintptr_t>(w->k) | reinterpret_cast<uintptr_t>(w->v) | reinterpret_cast<uintptr_t>(c.data);
  for (int i = 0; i < 3; ++i) al |= (uint64_t)w->k_strides[i] | (uint64_t)w->v_strides[i] | (uint64_t)c.strides[i];
  AF_REQUIRE((al & 15) == 0, what + "addresses and strides must be multiples of 16 bytes");
  RowArgs a;
  a.k = static_cast<const char*>(w->k), a.v = static_cast<const char*>(w->v);
  a.k_out = static_cast<char*>(w->k), a.v_out = static_cast<char*>(w->v);
  a.kl = w->k_strides[0], a.kn = w->k_strides[1], a.kh = w->k_strides[2];
  a.vl = w->v_strides[0], a.vn = w->v_strides[1], a.vh = w->v_strides[2];
  a.data = static_cast<char*>(c.data);
  a.dl = c.strides[0], a.dp = c.strides[1], a.dh = c.strides[2];
  a.slots = w->slots;
  a.rows = w->rows;
  a.n_rows = w->n_rows;
  a.count = w->count;
  a.n_slots = c.pages * c.page_size;
  a.layers = (int)c.layers;
  a.page = (int)c.page_size;
  a.heads = (int)c.heads;
  a.status = status;
  AF_REQUIRE(a.count <= 0x7fffffff && a.count * ceil_div(c.head_dim / 4 * a.heads, 32) <= 0x7fffffff, what + "too many rows");
  cudaStream_t s = as_stream(stream);
  const bool bf16 = c.dtype == AF_DTYPE_BF16;
  if (c.head_dim == 128) bf16 ? launch<AF_DTYPE_BF16, 128, WRITE>(a, s) : launch<AF_DTYPE_F16, 128, WRITE>(a, s);
  else bf16 ? launch<AF_DTYPE_BF16, 64, WRITE>(a, s) : launch<AF_DTYPE_F16, 64, WRITE>(a, s);
  return check_launch(name);
}

}  // namespace
}  // namespace kv4
}  // namespace af

using namespace af;

extern "C" int af_write_cache_int4(const af_int4_rows* w, uint32_t* status, void* stream) {
  return kv4::rows_call<true>(w, status, stream, "af_write_cache_int4");
}

extern "C" int af_read_cache_int4(const af_int4_rows* w, uint32_t* status, void* stream) {
  return kv4::rows_call<false>(w, status, stream, "af_read_cache_int4");
}
