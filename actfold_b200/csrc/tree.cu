// Index operators of a tree verification step over a paged key/value cache
// (sm_100a): block tables and slot maps, ancestor masks, acceptance of a
// drafted path, and the rows written into the cache. All of them are bound by
// launch and memory latency at serving sizes except large cache writes (HBM).
#include "tree.cuh"

namespace af {

namespace {

constexpr int kMaskThreads = 128;

// The nodes [s0, s0 + n) of tree b, or n = 0 (and the status bit) when starts is out of order or out of range.
__device__ __forceinline__ int tree_range(const int* __restrict__ starts, int b, int64_t total, int64_t most, unsigned* status, int* n) {
  const int s0 = starts[b], s1 = starts[b + 1];
  if (s0 < 0 || s1 < s0 || s1 > total || s1 - s0 > most) {
    if (threadIdx.x == 0 && status) atomicOr(status, AF_STATUS_BOUNDS);
    *n = 0;
    return 0;
  }
  *n = s1 - s0;
  return s0;
}

// mask[i] = {i} with every ancestor of i, position[i] = base + depth(i).
//
// CTA (c, b) takes nodes [128 c, 128 c + 128) of tree b with the parents of
// all nodes before them in shared memory, a thread per node. A parent comes
// before its children, so a walk to the root meets falling node numbers: the
// thread holds one 32-bit word of its row at a time and writes it when the walk
// leaves it. Rows of up to 32 words are put together in shared memory and
// leave in whole lines; wider ones go straight out. Bound by latency (starts, then
// parents, then the walk): 35726 nodes of 128 trees, 16 words each, take 8.0 to 8.6 us (10.0 us
// with rows stored straight out and parents loaded one after another), one tree of 26 nodes 2.9 to 3.3 us.
template <bool STAGED>
__global__ void __launch_bounds__(kMaskThreads) k_tree_masks(const int* __restrict__ parents, const int* __restrict__ starts,
                                                             int64_t total, int words, const int* __restrict__ base,
                                                             uint32_t* __restrict__ mask, int* __restrict__ positions,
                                                             unsigned* status) {
  extern __shared__ int sp[];
  __shared__ uint32_t rows[STAGED ? kMaskThreads * 33 : 1];  // a word more per row: no two lanes in one bank
  const int b = blockIdx.y, first = blockIdx.x * kMaskThreads;
  int n;
  const int s0 = tree_range(starts, b, total, 32 * (int64_t)words, status, &n);
  if (first >= n) return;
  const int last = min(n, first + kMaskThreads);
  for (int i0 = threadIdx.x; i0 < last; i0 += 4 * kMaskThreads) {
    int p[4];  // four loads at a time
#pragma unroll
    for (int u = 0; u < 4; ++u) p[u] = i0 + u * kMaskThreads < last ? parents[s0 + i0 + u * kMaskThreads] : -1;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = i0 + u * kMaskThreads;
      if (i >= last) break;
      if (p[u] < -1 || p[u] >= i) {
        if (status) atomicOr(status, AF_STATUS_BOUNDS);
        p[u] = -1;
      }
      sp[i] = p[u];
    }
  }
  __syncthreads();
  const int i = first + threadIdx.x;
  if (i < last) {
    uint32_t* row = STAGED ? rows + threadIdx.x * 33 : mask + (int64_t)(s0 + i) * words;
    int w = i >> 5, depth = 0;
    for (int z = words - 1; z > w; --z) row[z] = 0u;
    uint32_t bits = 1u << (i & 31);
    for (int p = sp[i]; p >= 0; p = sp[p]) {
      const int pw = p >> 5;
      while (pw != w) {
        row[w--] = bits;
        bits = 0u;
      }
      bits |= 1u << (p & 31);
      ++depth;
    }
    for (; w >= 0; --w) {
      row[w] = bits;
      bits = 0u;
    }
    positions[s0 + i] = depth + (base ? base[b] : 0);
  }
  if (STAGED) {
    __syncthreads();
    uint32_t* out = mask + (int64_t)(s0 + first) * words;
    for (int x = threadIdx.x; x < (last - first) * words; x += kMaskThreads) {
      const int r = x / words;
      out[x] = rows[r * 33 + (x - r * words)];
    }
  }
}

constexpr int kAcceptThreads = 256;

// The accepted path of tree b (a CTA per tree). link[i] is node i's parent
// where its token is the one wanted after that parent, -2 where it is not; a
// node is accepted when the walk along the links ends at a tree's top (-1).
// The deepest accepted node, of several the first, ends the path. Bound by
// latency (starts, parents, targets, walk): 4.4 us for 256 trees of 30 to 250
// nodes, 3.4 us for one of 26.
__global__ void __launch_bounds__(kAcceptThreads) k_accept_tree(const int* __restrict__ parents, const int64_t* __restrict__ tokens,
                                                                const int64_t* __restrict__ targets, const int* __restrict__ starts,
                                                                int64_t total, int64_t most, const int64_t* __restrict__ root_targets,
                                                                int keep, int* __restrict__ rows, int* __restrict__ counts,
                                                                int64_t* __restrict__ next, unsigned* status) {
  extern __shared__ int link[];
  __shared__ unsigned long long best_of[kAcceptThreads / 32];
  const int b = blockIdx.x;
  int n;
  const int s0 = tree_range(starts, b, total, most, status, &n);
  const int64_t root = root_targets ? root_targets[b] : -1;
  for (int i = threadIdx.x; i < n; i += kAcceptThreads) {
    int p = parents[s0 + i];
    const int64_t token = tokens[s0 + i];
    if (p < -1 || p >= i) {
      if (status) atomicOr(status, AF_STATUS_BOUNDS);
      p = -2;
    } else if (p >= 0) {
      if (token != targets[s0 + p]) p = -2;
    } else if (root_targets && token != root) {
      p = -2;
    }
    link[i] = p;
  }
  __syncthreads();
  // (depth, first node) as one number: the larger depth wins, then the smaller index.
  unsigned long long best = 0;
  for (int i = threadIdx.x; i < n; i += kAcceptThreads) {
    int p = link[i], depth = 1;
    while (p >= 0) {
      p = link[p];
      ++depth;
    }
    const unsigned long long key = ((unsigned long long)depth << 32) | (0xffffffffu - (unsigned)i);
    if (p == -1 && key > best) best = key;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
  if ((threadIdx.x & 31) == 0) best_of[threadIdx.x >> 5] = best;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kAcceptThreads / 32; ++w) best = max(best, best_of[w]);
  const int depth = (int)(best >> 32), count = min(depth, keep);
  int* out = rows + (int64_t)b * keep;
  for (int d = count + threadIdx.x; d < keep; d += kAcceptThreads) out[d] = -1;
  if (threadIdx.x == 0) {
    int64_t following = root;
    if (depth > 0) {
      int node = (int)(0xffffffffu - (unsigned)best);
      for (int d = depth - 1; d >= 0; --d) {
        if (d < keep) out[d] = s0 + node;
        if (d == count - 1) following = targets[s0 + node];
        node = link[node];
      }
    }
    counts[b] = count;
    next[b] = following;
  }
}

constexpr int kTableThreads = 1024;

struct TableArgs {
  int* tables;
  int64_t t_ld;
  int max_pages;
  const int *held, *lengths, *grow;
  int batch;
  int* ring;
  int64_t pool;
  const int64_t* range;
  int page;
  int64_t capacity;  // slots: packed, or per_request for each request
  int per_request;
  int *starts, *totals;
  int64_t* slots;
  int64_t* range_out;
  unsigned* status;
};

// Largest r with edge[r] <= x, for edge[0] = 0 <= ... and x < edge[batch].
__device__ __forceinline__ int request_of(const int* edge, int batch, int x) {
  int lo = 0, hi = batch;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (edge[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Block tables and slots. Every CTA scans all requests (three sums: pages
// taken, pages given back, new tokens) into shared memory, then the CTAs
// share the flat lists of taken pages, returned pages and slots, so one long
// prompt is spread like many short ones. Nothing that a CTA reads is written
// by another one: taken entries lie behind the held ones of their row, a slot
// in a taken page reads the ring, and the ring's places for returned pages
// are no free ones (returned <= held = pool - free). Bound by latency (lengths, the
// scan, the look through what changes hands, a search per slot) and by 64-bit divisions per page and slot: 14.7 us for
// 1000 requests with 84700 new tokens, 2613 pages taken and 3832 returned (0.8 MB, 0.1 us of HBM), 6.4 us for 5
// requests; without the look for negative entries 10.2 and 5.6 us, but then they would go round in the ring unseen.
__global__ void __launch_bounds__(kTableThreads) k_block_tables(const TableArgs a) {
  extern __shared__ int sh[];
  const int B = a.batch, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int* s_take = sh;              // [B + 1] exclusive sums
  int* s_give = sh + (B + 1);    // [B + 1]
  int* s_tok = sh + 2 * (B + 1); // [B + 1]
  __shared__ int64_t part[3][32];
  __shared__ unsigned s_bad;
  __shared__ int s_lost;
  if (tid == 0) s_bad = s_lost = 0;
  __syncthreads();
  int64_t run[3] = {0, 0, 0};
  unsigned bad = 0;
  for (int r0 = 0; r0 < B; r0 += kTableThreads) {
    const int r = r0 + tid;
    int64_t v[3] = {0, 0, 0};
    if (r < B) {
      const int64_t kept = a.lengths[r], held = a.held ? a.held[r] : kept, more = a.grow[r];
      if (kept < 0 || held < 0 || more < 0) {
        bad |= AF_STATUS_BOUNDS;
      } else {
        const int64_t had = (held + a.page - 1) / a.page, want = (kept + more + a.page - 1) / a.page;
        if (had > a.max_pages || want > a.max_pages || kept + more > 0x7fffffff || (a.per_request && more > a.per_request))
          bad |= AF_STATUS_CAPACITY;
        v[0] = max((int64_t)0, want - had);
        v[1] = max((int64_t)0, had - want);
        v[2] = more;
      }
    }
    int64_t inc[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      inc[k] = v[k];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, inc[k], o);
        if (lane >= o) inc[k] += y;
      }
      if (lane == 31) part[k][warp] = inc[k];
    }
    __syncthreads();
    if (warp < 3) {
      int64_t y = part[warp][lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t z = __shfl_up_sync(0xffffffffu, y, o);
        if (lane >= o) y += z;
      }
      part[warp][lane] = y;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      const int64_t before = run[k] + (warp ? part[k][warp - 1] : 0) + inc[k] - v[k];
      if (r < B) sh[k * (B + 1) + r] = (int)before;
      run[k] += part[k][31];
    }
    __syncthreads();
  }
  const int64_t head = a.range[0], tail = a.range[1];
  if (head < 0 || tail < head || tail - head > a.pool) bad |= AF_STATUS_BOUNDS;
  else if (run[0] > tail - head || run[1] > a.pool - (tail - head)) bad |= AF_STATUS_CAPACITY;
  if ((!a.per_request && run[2] > a.capacity) || run[2] > 0x7fffffff) bad |= AF_STATUS_CAPACITY;
  if (bad) atomicOr(&s_bad, bad);
  if (tid == 0) {
    s_take[B] = (int)min(run[0], (int64_t)0x7fffffff);
    s_give[B] = (int)min(run[1], (int64_t)0x7fffffff);
    s_tok[B] = (int)min(run[2], (int64_t)0x7fffffff);
  }
  __syncthreads();
  if (s_bad == 0) {
    // A negative entry among those that change hands is no page: it would come into a table, or into the ring and out of it
    // again. Every CTA looks through all of them before it writes (no CTA writes any of them), so all find the same.
    // Four loads at a time; of the returned ones a thread looks at neighbours, so that it searches for a request about once.
    const uint32_t take = s_take[B], give = s_give[B], pool = (uint32_t)a.pool;
    const uint32_t first = head < (1LL << 32) ? (uint32_t)head % pool : (uint32_t)(head % a.pool);
    int lost = 0;  // negative where one of them is
    for (uint32_t x = tid; x < take; x += 4 * kTableThreads) {
#pragma unroll
      for (uint32_t u = 0; u < 4 * kTableThreads; u += kTableThreads) {
        const uint32_t at = first + x + u;
        if (x + u < take) lost |= a.ring[at < pool ? at : at - pool];
      }
    }
    const uint32_t each = (give + kTableThreads - 1) / kTableThreads, end = min(give, (tid + 1) * each);
    for (uint32_t x = tid * each; x < end;) {
      const int r = request_of(s_give, B, (int)x);
      const uint32_t stop = min(end, (uint32_t)s_give[r + 1]), want = ((uint32_t)a.lengths[r] + a.grow[r] + a.page - 1) / (uint32_t)a.page;
      const int* row = a.tables + r * a.t_ld + want - s_give[r];
      for (; x < stop; x += 4) {
#pragma unroll
        for (uint32_t u = 0; u < 4; ++u)
          if (x + u < stop) lost |= row[x + u];
      }
      x = stop;
    }
    if (lost < 0) s_lost = 1;
  }
  __syncthreads();
  const bool ok = s_bad == 0 && s_lost == 0;
  if (blockIdx.x == 0) {
    for (int r = tid; r <= B; r += kTableThreads) a.starts[r] = ok ? s_tok[r] : 0;
    for (int r = tid; r < B; r += kTableThreads) a.totals[r] = ok ? a.lengths[r] + a.grow[r] : (a.held ? a.held[r] : a.lengths[r]);
    if (tid == 0) {
      a.range_out[0] = ok ? head + run[0] : head;
      a.range_out[1] = ok ? tail + run[1] : tail;
      if (!ok && a.status) atomicOr(a.status, s_bad ? s_bad : AF_STATUS_BOUNDS);
    }
  }
  const int64_t me = (int64_t)blockIdx.x * kTableThreads + tid, step = (int64_t)gridDim.x * kTableThreads;
  if (ok) {
    for (int64_t x = me; x < s_take[B]; x += step) {
      const int r = request_of(s_take, B, (int)x);
      const int held = a.held ? a.held[r] : a.lengths[r];
      a.tables[r * a.t_ld + (held + (int64_t)a.page - 1) / a.page + (x - s_take[r])] = a.ring[(head + x) % a.pool];
    }
    for (int64_t x = me; x < s_give[B]; x += step) {
      const int r = request_of(s_give, B, (int)x);
      const int64_t want = ((int64_t)a.lengths[r] + a.grow[r] + a.page - 1) / a.page;
      a.ring[(tail + x) % a.pool] = a.tables[r * a.t_ld + want + (x - s_give[r])];
    }
  }
  for (int64_t x = me; x < a.capacity; x += step) {
    int64_t slot = -1;
    int r = -1, i = 0;
    if (ok && a.per_request) {
      r = (int)(x / a.per_request);
      i = (int)(x - (int64_t)r * a.per_request);
      if (i >= s_tok[r + 1] - s_tok[r]) r = -1;
    } else if (ok && x < s_tok[B]) {
      r = request_of(s_tok, B, (int)x);
      i = (int)x - s_tok[r];
    }
    if (r >= 0) {
      const int64_t kept = a.lengths[r], held = a.held ? a.held[r] : kept, pos = kept + i;
      const int64_t k = pos / a.page, had = (held + a.page - 1) / a.page;
      const int page = k < had ? a.tables[r * a.t_ld + k] : a.ring[(head + s_take[r] + (k - had)) % a.pool];
      if (page >= 0) slot = (int64_t)page * a.page + (pos - k * a.page);
      else if (a.status) atomicOr(a.status, AF_STATUS_BOUNDS);  // a held entry that is no page
    }
    a.slots[x] = slot;
  }
}

struct WriteArgs {
  const char *k, *v;
  int64_t kl, kn, kh, vl, vn, vh;  // byte strides of the rows: layer, row, head
  char *kc, *vc;
  int64_t kcl, kcp, kct, kch, vcl, vcp, vct, vch;  // of the caches: layer, page, token, head
  const int64_t* slots;
  const int* rows;
  int64_t n_rows, count, n_slots;
  int layers, page, heads;
  int per_head;  // vectors (or bytes) of a head
  unsigned* status;
};

constexpr int kWriteThreads = 256;

// A warp moves 32 U vectors of (keys, then values) of one row: U 16-byte loads
// per lane in flight, then U stores. Bound by HBM (every byte is read and written
// once): 10391 rows of 32 heads x 128 bf16, keys and values, take 53.5 us (6.37 TB/s);
// with U = 4 and 64-bit divisions they took 64 us, with U = 8 and 32-bit ones 56. FLAT: a row's heads lie
// next to one another on both sides, so there is no head to divide for.
template <typename V, int U, bool FLAT>
__global__ void __launch_bounds__(kWriteThreads) k_write_cache(const WriteArgs a, int chunks) {
  const int lane = threadIdx.x & 31;
  const int item = blockIdx.x * (kWriteThreads / 32) + (threadIdx.x >> 5);  // (row, chunk)
  const int m = item / chunks, chunk = item - m * chunks, l = blockIdx.y;
  if (m >= a.count) return;
  const int64_t slot = a.slots[m];
  const int64_t row = a.rows ? a.rows[m] : m;
  if (slot < 0 || row < 0) return;
  if (slot >= a.n_slots || row >= a.n_rows) {
    if (lane == 0 && a.status) atomicOr(a.status, AF_STATUS_BOUNDS);
    return;
  }
  const int64_t pg = slot < 0x7fffffff ? (int)slot / a.page : slot / a.page, t = slot - pg * a.page;
  const int half = a.heads * a.per_head;
  const char* k = a.k + l * a.kl + row * a.kn;
  const char* v = a.v + l * a.vl + row * a.vn;
  char* kc = a.kc + l * a.kcl + pg * a.kcp + t * a.kct;
  char* vc = a.vc + l * a.vcl + pg * a.vcp + t * a.vct;
  const int x0 = chunk * 32 * U + lane;
  V buf[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int x = x0 + 32 * u;
    if (x < 2 * half) {
      const bool val = x >= half;
      const int y = val ? x - half : x, h = FLAT ? 0 : y / a.per_head, c = y - h * a.per_head;
      buf[u] = reinterpret_cast<const V*>((val ? v : k) + h * (val ? a.vh : a.kh))[c];
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int x = x0 + 32 * u;
    if (x < 2 * half) {
      const bool val = x >= half;
      const int y = val ? x - half : x, h = FLAT ? 0 : y / a.per_head, c = y - h * a.per_head;
      reinterpret_cast<V*>((val ? vc : kc) + h * (val ? a.vch : a.kch))[c] = buf[u];
    }
  }
}

template <typename V, int U>
void launch_write(const WriteArgs& a, cudaStream_t s) {
  const int chunks = (int)ceil_div(2 * (int64_t)a.heads * a.per_head, 32 * U);
  const dim3 grid((unsigned)ceil_div((int64_t)chunks * a.count, kWriteThreads / 32), (unsigned)a.layers);
  const int64_t head = (int64_t)a.per_head * sizeof(V);
  if (a.heads == 1 || (a.kh == head && a.vh == head && a.kch == head && a.vch == head)) k_write_cache<V, U, true><<<grid, kWriteThreads, 0, s>>>(a, chunks);
  else k_write_cache<V, U, false><<<grid, kWriteThreads, 0, s>>>(a, chunks);
}

// Without this a kernel gets 48 KB, its static shared memory (up to 1 KB here) among them. `most` is what any call can
// need, the same each time: a call on another thread cannot lower it between this one's limit and its launch.
template <typename K>
int allow_smem(K kernel, size_t bytes, size_t most, const char* what) {
  if (bytes <= 47 * 1024) return AF_OK;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
  if (e != cudaSuccess) return fail(AF_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
  return AF_OK;
}

}  // namespace
}  // namespace af

using namespace af;

extern "C" int af_tree_masks(const int32_t* parents, const int32_t* starts, int64_t batch, int64_t total, int64_t words,
                             const int32_t* base, int32_t* mask, int32_t* positions, uint32_t* status, void* stream) {
  AF_REQUIRE(batch >= 0 && total >= 0 && words > 0, "af_tree_masks: bad shape");
  AF_REQUIRE(batch <= 65535 && words <= AF_TREE_MAX_NODES / 32, "af_tree_masks: at most 65535 trees of 16384 nodes");
  AF_REQUIRE(total <= 0x7fffffff, "af_tree_masks: node numbers are 32 bits wide");
  if (batch == 0 || total == 0) return AF_OK;
  AF_REQUIRE(parents && starts && mask && positions, "af_tree_masks: null pointer");
  const int64_t most = words * 32 < total ? words * 32 : total;
  const size_t smem = (size_t)most * sizeof(int);
  const auto kernel = words <= 32 ? k_tree_masks<true> : k_tree_masks<false>;
  if (words > 32)  // (up to 32 words: 4 KB of parents)
    if (int st = allow_smem(kernel, smem, AF_TREE_MAX_NODES * sizeof(int), "af_tree_masks")) return st;
  kernel<<<dim3((unsigned)ceil_div(most, kMaskThreads), (unsigned)batch), kMaskThreads, smem, as_stream(stream)>>>(
      parents, starts, total, (int)words, base, reinterpret_cast<uint32_t*>(mask), positions, status);
  return check_launch("af_tree_masks");
}

extern "C" int af_accept_tree(const int32_t* parents, const int64_t* tokens, const int64_t* targets, const int32_t* starts,
                              int64_t batch, int64_t total, int64_t max_nodes, const int64_t* root_targets, int64_t keep,
                              int32_t* rows, int32_t* counts, int64_t* next_tokens, uint32_t* status, void* stream) {
  AF_REQUIRE(batch >= 0 && total >= 0 && max_nodes >= 0 && keep > 0, "af_accept_tree: bad shape");
  AF_REQUIRE(max_nodes <= AF_TREE_MAX_NODES && keep <= AF_TREE_MAX_NODES, "af_accept_tree: at most 16384 nodes per tree");
  AF_REQUIRE(total <= 0x7fffffff && batch <= 0x7fffffff, "af_accept_tree: node numbers are 32 bits wide");
  if (batch == 0) return AF_OK;
  AF_REQUIRE(starts && rows && counts && next_tokens, "af_accept_tree: null pointer");
  AF_REQUIRE(total == 0 || (parents && tokens && targets), "af_accept_tree: null pointer");
  const int64_t most = max_nodes < total ? max_nodes : total;
  const size_t smem = (size_t)most * sizeof(int);
  if (int st = allow_smem(k_accept_tree, smem, AF_TREE_MAX_NODES * sizeof(int), "af_accept_tree")) return st;
  k_accept_tree<<<(unsigned)batch, kAcceptThreads, smem, as_stream(stream)>>>(parents, tokens, targets, starts, total, most, root_targets,
                                                                            (int)keep, rows, counts, next_tokens, status);
  return check_launch("af_accept_tree");
}

extern "C" int af_block_tables(int32_t* tables, int64_t tables_stride, int64_t max_pages, const int32_t* held, const int32_t* lengths,
                               const int32_t* grow, int64_t batch, int32_t* free_pages, int64_t pool, const int64_t* free_range,
                               int64_t page_size, int64_t slot_capacity, int64_t slots_per_request, int32_t* starts, int32_t* totals,
                               int64_t* slots, int64_t* free_range_out, uint32_t* status, void* stream) {
  AF_REQUIRE(batch > 0 && max_pages >= 0 && pool > 0 && page_size > 0 && slot_capacity >= 0 && slots_per_request >= 0,
             "af_block_tables: bad shape");
  AF_REQUIRE(batch <= AF_TABLES_MAX_BATCH, "af_block_tables: at most 16384 requests");
  AF_REQUIRE(max_pages <= 0x7fffffff && pool <= 0x7fffffff && page_size <= (1 << 20) && slot_capacity <= 0x7fffffff,
             "af_block_tables: size too large");
  AF_REQUIRE(slots_per_request == 0 || slot_capacity == batch * slots_per_request,
             "af_block_tables: slot_capacity must be batch * slots_per_request");
  AF_REQUIRE(lengths && grow && free_pages && free_range && starts && totals && free_range_out && (tables || max_pages == 0) &&
                 (slots || slot_capacity == 0),
             "af_block_tables: null pointer");
  AF_REQUIRE(free_range != free_range_out, "af_block_tables: the new range needs a place of its own");
  TableArgs a;
  a.tables = tables;
  a.t_ld = tables_stride;
  a.max_pages = (int)max_pages;
  a.held = held;
  a.lengths = lengths;
  a.grow = grow;
  a.batch = (int)batch;
  a.ring = free_pages;
  a.pool = pool;
  a.range = free_range;
  a.page = (int)page_size;
  a.capacity = slot_capacity;
  a.per_request = (int)slots_per_request;
  a.starts = starts;
  a.totals = totals;
  a.slots = slots;
  a.range_out = free_range_out;
  a.status = status;
  const size_t smem = 3 * (size_t)(batch + 1) * sizeof(int);
  if (int st = allow_smem(k_block_tables, smem, 3 * (AF_TABLES_MAX_BATCH + 1) * sizeof(int), "af_block_tables")) return st;
  // A thread writes about two slots; returned pages count as well, where requests end.
  const int64_t want = ceil_div(slot_capacity + batch * max_pages / 16, 2 * kTableThreads);
  const int sms = sm_count();
  const unsigned blocks = (unsigned)(want < 1 ? 1 : want > sms ? sms : want);
  k_block_tables<<<blocks, kTableThreads, smem, as_stream(stream)>>>(a);
  return check_launch("af_block_tables");
}

extern "C" int af_write_cache(const af_cache_rows* w, uint32_t* status, void* stream) {
  AF_REQUIRE(w, "af_write_cache: null pointer");
  AF_REQUIRE(w->layers >= 0 && w->n_rows >= 0 && w->count >= 0 && w->pages >= 0 && w->page_size > 0 && w->heads >= 0 && w->head_bytes >= 0,
             "af_write_cache: bad shape");
  if (w->layers == 0 || w->count == 0 || w->heads == 0 || w->head_bytes == 0) return AF_OK;
  AF_REQUIRE(w->slots && (w->n_rows == 0 || (w->k && w->v)) && (w->pages == 0 || (w->k_cache && w->v_cache)),
             "af_write_cache: null pointer");  // (of no rows or no pages every entry is skipped)
  AF_REQUIRE(w->heads <= (1 << 20) && w->head_bytes <= (1 << 20) && w->heads * w->head_bytes <= (1 << 28) && w->page_size <= (1 << 20) &&
                 w->layers <= 0x7fffffff,
             "af_write_cache: size too large");
  WriteArgs a;
  a.k = static_cast<const char*>(w->k);
  a.v = static_cast<const char*>(w->v);
  a.kc = static_cast<char*>(w->k_cache);
  a.vc = static_cast<char*>(w->v_cache);
  a.kl = w->k_strides[0], a.kn = w->k_strides[1], a.kh = w->k_strides[2];
  a.vl = w->v_strides[0], a.vn = w->v_strides[1], a.vh = w->v_strides[2];
  a.kcl = w->k_cache_strides[0], a.kcp = w->k_cache_strides[1], a.kct = w->k_cache_strides[2], a.kch = w->k_cache_strides[3];
  a.vcl = w->v_cache_strides[0], a.vcp = w->v_cache_strides[1], a.vct = w->v_cache_strides[2], a.vch = w->v_cache_strides[3];
  a.slots = w->slots;
  a.rows = w->rows;
  a.n_rows = w->n_rows;
  a.count = w->count;
  a.n_slots = w->pages * w->page_size;
  a.layers = (int)w->layers;
  a.page = (int)w->page_size;
  a.heads = (int)w->heads;
  a.status = status;
  uint64_t al = reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v) | reinterpret_cast<uintptr_t>(a.kc) |
                reinterpret_cast<uintptr_t>(a.vc) | (uint64_t)w->head_bytes;
  for (int i = 0; i < 3; ++i) al |= (uint64_t)w->k_strides[i] | (uint64_t)w->v_strides[i];
  for (int i = 0; i < 4; ++i) al |= (uint64_t)w->k_cache_strides[i] | (uint64_t)w->v_cache_strides[i];
  const int unit = (al & 15) == 0 ? 16 : (al & 3) == 0 ? 4 : 1;
  a.per_head = (int)(w->head_bytes / unit);
  AF_REQUIRE(a.layers <= 65535 && a.count * ceil_div(2 * (int64_t)a.heads * a.per_head, 128) <= 0x7fffffff, "af_write_cache: too many rows");
  cudaStream_t s = as_stream(stream);
  if (unit == 16 && a.heads * a.per_head >= 256) launch_write<uint4, 8>(a, s);
  else if (unit == 16) launch_write<uint4, 4>(a, s);
  else if (unit == 4) launch_write<uint32_t, 4>(a, s);
  else launch_write<uint8_t, 4>(a, s);
  return check_launch("af_write_cache");
}
