// Attention of drafted trees over a paged key/value cache (sm_100a).
#include "tree.cuh"

namespace af {

namespace {

template <int DT>
__device__ __forceinline__ uint16_t to_bits(float x) {
  if constexpr (DT == AF_DTYPE_BF16) return f2bf_bits(x);
  else {
    const __half h = __float2half_rn(x);
    return *reinterpret_cast<const uint16_t*>(&h);
  }
}

// A warp per (node, query head): lane x holds dims x, x + 32, ... of the
// query and of the sum, keys come one at a time.
template <int DT, int HD>
__global__ void __launch_bounds__(256) k_tree_attention_rows(const af_tree_attention_args a, unsigned* status) {
  const int lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int64_t node = item / a.n_heads;
  const int h = (int)(item % a.n_heads);
  if (item == 0) {
    for (int b = lane; b < a.batch; b += 32)
      if ((a.starts[b] < 0 || a.starts[b] > a.starts[b + 1] || a.starts[b + 1] > a.total) && status) atomicOr(status, AF_STATUS_BOUNDS);
  }
  if (node >= a.total || node >= a.starts[a.batch]) return;
  int lo = 0, hi = (int)a.batch;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.starts[mid] <= node) lo = mid;
    else hi = mid;
  }
  const int b = lo, s0 = a.starts[b], n = a.starts[b + 1] - s0, i = (int)node - s0;
  const int64_t t = a.lengths[b];
  if (s0 < 0 || i < 0 || i >= n || s0 + (int64_t)n > a.total || (a.mask && n > 32 * a.words) || t < 0 || t > a.max_pages * a.page_size) {
    if (lane == 0 && status) atomicOr(status, AF_STATUS_BOUNDS);
    return;
  }
  const int kvh = h / (int)(a.n_heads / a.n_kv_heads);
  constexpr int R = HD / 32;
  float q[R], acc[R], m = -INFINITY, l = 0.f;
  const char* qp = static_cast<const char*>(a.q) + node * a.q_strides[0] + h * a.q_strides[1];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    q[r] = load_scalar<DT>(qp, lane + 32 * r) * (float)a.scale;
    acc[r] = 0.f;
  }
  for (int64_t j = 0; j < t + n; ++j) {
    const char *kp, *vp;
    if (j < t) {
      const int64_t pg = a.tables[b * a.tables_stride + j / a.page_size], off = j % a.page_size;
      if (pg < 0 || pg >= a.pages) {
        if (lane == 0 && status) atomicOr(status, AF_STATUS_BOUNDS);
        continue;
      }
      kp = static_cast<const char*>(a.k_cache) + pg * a.k_cache_strides[0] + off * a.k_cache_strides[1] + kvh * a.k_cache_strides[2];
      vp = static_cast<const char*>(a.v_cache) + pg * a.v_cache_strides[0] + off * a.v_cache_strides[1] + kvh * a.v_cache_strides[2];
    } else {
      const int x = (int)(j - t);
      if (a.mask ? !((a.mask[node * a.mask_stride + (x >> 5)] >> (x & 31)) & 1) : x > i) continue;
      kp = static_cast<const char*>(a.k) + (s0 + x) * a.k_strides[0] + kvh * a.k_strides[1];
      vp = static_cast<const char*>(a.v) + (s0 + x) * a.v_strides[0] + kvh * a.v_strides[1];
    }
    float s = 0.f;
#pragma unroll
    for (int r = 0; r < R; ++r) s += q[r] * load_scalar<DT>(kp, lane + 32 * r);
    s = warp_sum(s);
    const float up = fmaxf(m, s);
    const float old = m == -INFINITY ? 0.f : expf(m - up), p = s == -INFINITY ? 0.f : expf(s - up);
    m = up;
    l = l * old + p;
#pragma unroll
    for (int r = 0; r < R; ++r) acc[r] = acc[r] * old + p * load_scalar<DT>(vp, lane + 32 * r);
  }
  char* op = static_cast<char*>(a.out) + node * a.out_strides[0] + h * a.out_strides[1];
#pragma unroll
  for (int r = 0; r < R; ++r) reinterpret_cast<uint16_t*>(op)[lane + 32 * r] = to_bits<DT>(l > 0.f ? acc[r] / l : acc[r]);
  if (lane == 0 && a.lse) a.lse[node * a.n_heads + h] = l > 0.f ? m + logf(l) : (l == l ? -INFINITY : l);
}

int64_t workspace_bytes() { return 256; }

int check_args(const af_tree_attention_args& a) {
  AF_REQUIRE(a.batch >= 0 && a.total >= 0 && a.max_pages >= 0 && a.pages >= 0, "af_tree_attention: bad shape");
  AF_REQUIRE(a.n_heads > 0 && a.n_kv_heads > 0 && a.n_heads % a.n_kv_heads == 0, "af_tree_attention: n_heads must be a multiple of n_kv_heads");
  AF_REQUIRE(a.n_heads / a.n_kv_heads <= 64, "af_tree_attention: at most 64 query heads per key/value head");
  AF_REQUIRE(a.head_dim == 64 || a.head_dim == 128, "af_tree_attention: head_dim must be 64 or 128");
  AF_REQUIRE(a.dtype == AF_DTYPE_F16 || a.dtype == AF_DTYPE_BF16, "af_tree_attention: dtype must be fp16 or bf16");
  AF_REQUIRE(a.page_size > 0 && a.page_size % 8 == 0 && a.page_size <= (1 << 20), "af_tree_attention: page_size must be a multiple of 8");
  AF_REQUIRE(a.batch <= AF_TREE_ATTN_MAX_BATCH, "af_tree_attention: at most 16384 requests");
  AF_REQUIRE(a.total <= (1 << 28) && a.pages <= 0x7fffffff && a.n_heads <= (1 << 16) && a.max_pages * a.page_size <= 0x7fffffff,
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
  AF_REQUIRE(a.workspace_bytes >= workspace_bytes(), "af_tree_attention: the workspace is too small");
  AF_REQUIRE((al & 15) == 0, "af_tree_attention: addresses and strides must be multiples of 16 bytes");
  return AF_OK;
}

}  // namespace
}  // namespace af

using namespace af;

extern "C" int af_tree_attention_workspace_bytes(int64_t* bytes) {
  AF_REQUIRE(bytes, "af_tree_attention_workspace_bytes: null pointer");
  *bytes = workspace_bytes();
  return AF_OK;
}

extern "C" int af_tree_attention(const af_tree_attention_args* p, uint32_t* status, void* stream) {
  AF_REQUIRE(p, "af_tree_attention: null pointer");
  const af_tree_attention_args& a = *p;
  if (int st = check_args(a)) return st;
  if (a.batch == 0 || a.total == 0) return AF_OK;
  const unsigned blocks = (unsigned)ceil_div(a.total * a.n_heads, 8);
  cudaStream_t s = as_stream(stream);
  if (a.dtype == AF_DTYPE_BF16) {
    if (a.head_dim == 128) k_tree_attention_rows<AF_DTYPE_BF16, 128><<<blocks, 256, 0, s>>>(a, status);
    else k_tree_attention_rows<AF_DTYPE_BF16, 64><<<blocks, 256, 0, s>>>(a, status);
  } else {
    if (a.head_dim == 128) k_tree_attention_rows<AF_DTYPE_F16, 128><<<blocks, 256, 0, s>>>(a, status);
    else k_tree_attention_rows<AF_DTYPE_F16, 64><<<blocks, 256, 0, s>>>(a, status);
  }
  return check_launch("af_tree_attention");
}
