// Rows into and out of the 4-bit paged cache (sm_100a).
//
// Per token and head of 128 dims 512 bytes of 16-bit rows against 160 of the
// cache, so HBM bounds both kernels once the arithmetic is cheap enough: an SM has
// 27 cycles for the 256 values of that token and head. Writing: a lane takes
// the 32 dims of a pair (64 bytes), so that extremes, scale and reciprocal are
// found once for them. Reading: a lane takes 8 dims, a code word and 16 bytes out, of one
// head after the other.
//
// 10391 rows of 32 heads x 128: written in 65 us (the bytes need 34), bound by the dozen instructions that a value takes (a
// lane with 8 dims, and divisions for ties: 123 us; persistent CTAs that load ahead: 87 to 90); read in 41 us (the same bytes), by the cache's
// scattered rows of 64 and 16 bytes.
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

// Eight codes next to one another, as exact arithmetic rounds them.
template <int DT>
__device__ __noinline__ uint32_t careful_word(uint4 x, float offset, float scale) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  uint32_t word = 0;
#pragma unroll 1
  for (int i = 0; i < 8; ++i) {
    const float y = from16<DT>((w[i >> 1] >> (16 * (i & 1))) & 0xffffu);
    word |= careful_code(y, offset, y - offset, scale) << (4 * (i >> 1) + 16 * (i & 1));
  }
  return word;
}

// The 32 values of a pair into four code words.
template <int DT>
__device__ __forceinline__ uint4 encode(const uint4* x, uint32_t& pair) {
  using P = Pair16<DT>;
  auto lo2 = P::make(x[0].x), hi2 = lo2;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    lo2 = __hmin2_nan(lo2, __hmin2_nan(__hmin2_nan(P::make(x[i].x), P::make(x[i].y)), __hmin2_nan(P::make(x[i].z), P::make(x[i].w))));
    hi2 = __hmax2_nan(hi2, __hmax2_nan(__hmax2_nan(P::make(x[i].x), P::make(x[i].y)), __hmax2_nan(P::make(x[i].z), P::make(x[i].w))));
  }
  const float l0 = from16<DT>(bits_of(lo2) & 0xffffu), l1 = from16<DT>(bits_of(lo2) >> 16);
  const float h0 = from16<DT>(bits_of(hi2) & 0xffffu), h1 = from16<DT>(bits_of(hi2) >> 16);
  const float low = fminf(l0, l1), range = fmaxf(h0, h1) - low;
  const bool sound = !(isnan(l0) || isnan(l1)) && fabsf(range) <= 3.402823466e38f;
  if (!sound) {  // the group stands for NaN
    pair = (DT == AF_DTYPE_BF16 ? 0x7fc0u : 0x7e00u) << 16;
    return make_uint4(0, 0, 0, 0);
  }
  uint32_t s16 = to16<DT>(range / 15.f);
  if (!finite16<DT>(to16<DT>(fmaf(15.f, from16<DT>(s16), low)))) --s16;
  pair = s16 | to16<DT>(low) << 16;
  const float scale = from16<DT>(s16), half = 0.5f * scale;
  if (scale == 0.f) return make_uint4(0, 0, 0, 0);
  // A number below 2^22 added to 1.5 * 2^23 is rounded to a whole one, here to one of the two codes that x - offset lies between:
  // the reciprocal is not exact. What is left, r = x - offset - code * scale, is: less than half a step says that the code is the nearest.
  // Of normal values in bf16 0.2 % are a tie or beyond, so that 40 % of a warp's words take the longer way: there the other code is
  // taken where |r| is more than half a step, or is half a step and the code odd. (As whole numbers the magnitudes of floats are
  // in their order. All words the longer way: 73 us for the 10391 rows above.)
  constexpr float magic = 12582912.f;
  constexpr uint32_t magic_bits = 0x4b400000u;
  const float inv = 1.f / scale;
  const bool usual = inv <= 3.402823466e38f && range <= 15.25f * scale;  // else the scale has lost its precision, and codes may pass 15
  // Differences lose nothing of an offset that is 0 or not far below them: its last bit is worth 2^-10 of it or more, that of x - offset 2^-23
  // of the range at most.
  const bool near = low == 0.f || fabsf(low) >= range * (1.f / 8192.f);
  auto shift = [](int c) { return 4 * (c >> 1) + 16 * (c & 1); };
  uint32_t out[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
    auto value = [&](int c) { return from16<DT>(c & 1 ? w[c >> 1] >> 16 : w[c >> 1] & 0xffffu); };
    uint32_t word = 0u - magic_bits * 0x11111111u;  // (modulo 2^32, as the sums below)
    float off = 0.f;
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      const float d = value(c) - low, t = fmaf(d, inv, magic);
      off = fmaxf(off, fabsf(fmaf(magic - t, scale, d)));
      word += __float_as_uint(t) << shift(c);
    }
    if (!usual) {
      word = careful_word<DT>(x[i], low, scale);
    } else if (off >= half) {
      bool sure = near;
      word = 0;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const float y = value(c), d = y - low, t = fmaf(d, inv, magic), r = fmaf(magic - t, scale, d);
        sure &= low + d == y;  // (a tie is none where the difference has lost something in fp32: here of y)
        const uint32_t step = __float_as_int(fabsf(r)) + (__float_as_int(t) & 1) > __float_as_int(half) ? 1u | (__float_as_int(r) >> 31) : 0u;
        word += (__float_as_uint(t) - magic_bits + step) << shift(c);
      }
      if (!sure) word = careful_word<DT>(x[i], low, scale);
    }
    out[i] = word;
  }
  return make_uint4(out[0], out[1], out[2], out[3]);
}

// A thread takes the 32 dims of a pair, of a key or value of one head.
template <int DT, int HD>
__global__ void __launch_bounds__(kThreads) k_write(const RowArgs a) {
  using B = Block<HD>;
  constexpr int G = HD / kGroup;  // pairs of a row
  const uint32_t item = blockIdx.x * kThreads + threadIdx.x, per_row = 2 * G * a.heads;  // (below 2^31: checked by the host)
  const int m = (int)(item / per_row), x = (int)(item - m * per_row), l = blockIdx.y;
  if (m >= a.count) return;
  const int64_t slot = a.slots[m];
  const int64_t row = a.rows ? a.rows[m] : m;
  if (slot < 0 || row < 0) return;
  if (slot >= a.n_slots || row >= a.n_rows) {
    if (x == 0 && a.status) atomicOr(a.status, AF_STATUS_BOUNDS);
    return;
  }
  const int h = x / (2 * G), val = x / G % 2, g = x % G;
  const uint4* from = reinterpret_cast<const uint4*>((val ? a.v + l * a.vl + row * a.vn + h * a.vh : a.k + l * a.kl + row * a.kn + h * a.kh) + 64 * g);
  uint4 v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = from[i];
  const int64_t pg = slot < 0x7fffffff ? (int)slot / a.page : slot / a.page;
  const int t = (int)(slot - pg * a.page), r = t % kBlockTokens;
  char* part = a.data + l * a.dl + pg * a.dp + h * a.dh + (int64_t)(t / kBlockTokens) * B::kBytes + val * B::kPart;
  uint32_t pair;
  *reinterpret_cast<uint4*>(part + B::word(r, 4 * g)) = encode<DT>(v, pair);
  *reinterpret_cast<uint32_t*>(part + B::pair(r, g)) = pair;
}

// A warp takes U passes over one slot's heads: with 128 dims the 32 code words of a head's key and value, with 64 those of two heads.
template <int DT, int HD, int U>
__global__ void __launch_bounds__(kThreads) k_read(const RowArgs a, int chunks) {
  using B = Block<HD>;
  constexpr int W = HD / 8, H = 32 / (2 * W);  // words of a row; heads of a pass
  const int lane = threadIdx.x & 31;
  const int item = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);  // (row, chunk of heads)
  const int m = chunks == 1 ? item : item / chunks, chunk = item - m * chunks, l = blockIdx.y;
  if (m >= a.count) return;
  int64_t slot = a.slots[m];
  if (slot >= a.n_slots) {
    if (lane == 0 && a.status) atomicOr(a.status, AF_STATUS_BOUNDS);
    slot = -1;
  }
  const int64_t pg = slot < 0x7fffffff ? (int)slot / a.page : slot / a.page;
  const int t = (int)(slot - pg * a.page), r = t % kBlockTokens;
  const int h0 = chunk * U * H + lane / (2 * W), val = lane / W % 2, w = lane % W;
  const char* word_at = a.data + l * a.dl + pg * a.dp + h0 * a.dh + (int64_t)(t / kBlockTokens) * B::kBytes + val * B::kPart;
  const char* pair_at = word_at + B::pair(r, w / 4);
  word_at += B::word(r, w);
  const int64_t step = H * a.dh, oh = val ? a.vh : a.kh;
  char* to = (val ? a.v_out + l * a.vl + m * a.vn : a.k_out + l * a.kl + m * a.kn) + h0 * oh + 16 * w;
  uint32_t word[U], pair[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const bool there = slot >= 0 && h0 + u * H < a.heads;
    word[u] = there ? *reinterpret_cast<const uint32_t*>(word_at + u * step) : 0;
    pair[u] = there ? *reinterpret_cast<const uint32_t*>(pair_at + u * step) : 0;
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    // Word and pair are 0 where there is no slot, and so are the values.
    const uint32_t s2 = __byte_perm(pair[u], 0, 0x1010), o2 = __byte_perm(pair[u], 0, 0x3232);
    const uint4 y = make_uint4(two_values<DT, 0>(word[u], s2, o2), two_values<DT, 1>(word[u], s2, o2), two_values<DT, 2>(word[u], s2, o2),
                               two_values<DT, 3>(word[u], s2, o2));
    if (h0 + u * H < a.heads) *reinterpret_cast<uint4*>(to + u * (H * oh)) = y;
  }
}

template <int DT, int HD, bool WRITE>
void launch(const RowArgs& a, cudaStream_t s) {
  if constexpr (WRITE) {
    const dim3 grid((unsigned)ceil_div(a.count * 2 * (HD / kGroup) * a.heads, kThreads), (unsigned)a.layers);
    k_write<DT, HD><<<grid, kThreads, 0, s>>>(a);
  } else {
    // As many passes in flight as a row has, up to eight.
    const int passes = (int)ceil_div(a.heads, 128 / HD), u = passes > 4 ? 8 : passes > 2 ? 4 : passes > 1 ? 2 : 1;
    const int chunks = (int)ceil_div(passes, u);
    const dim3 grid((unsigned)ceil_div((int64_t)chunks * a.count, kThreads / 32), (unsigned)a.layers);
    if (u == 8) k_read<DT, HD, 8><<<grid, kThreads, 0, s>>>(a, chunks);
    else if (u == 4) k_read<DT, HD, 4><<<grid, kThreads, 0, s>>>(a, chunks);
    else if (u == 2) k_read<DT, HD, 2><<<grid, kThreads, 0, s>>>(a, chunks);
    else k_read<DT, HD, 1><<<grid, kThreads, 0, s>>>(a, chunks);
  }
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
  AF_REQUIRE(runs_apart(c, true), what + "the cache's strides let its entries share memory");
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
  AF_REQUIRE(a.count <= (1 << 28) && a.count * (2 * (c.head_dim / kGroup) * a.heads + 32) <= 0x7fffff00, what + "too many rows");
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
