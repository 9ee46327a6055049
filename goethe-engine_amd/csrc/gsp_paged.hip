// The paged cache around a verify round (include/gsp.h): the step of the bookkeeping (gsp_pages_step) and the move of the
// accepted paths (gsp_keep_path).
#include "gse_dev.h"
#include "gsp_int.h"

namespace gse {

namespace {

// ---- the step -----------------------------------------------------------------------------------------------------------
// Per request r: kept = length + keep (0 when keep < 0), need = ceil((kept + add) / page) pages of which it holds `held`. The
// exclusive sums over the requests of add, of the pages lacking and of the pages too many say where each request's new
// tokens start, which ring entries it takes and which it gives back to. A new page p (held <= p < need) holds a new token at
// its first place (kept <= held * page), so the thread of that token also writes the page into the table.
//
// Every workgroup forms the sums itself (16 bytes a request, from cache), RC requests at a time, so no workgroup waits for
// another; then it takes its share of the chunk's tokens and of the pages given back. The state is read from counters and
// written to counters_out by one workgroup: when they are the same array, by a second launch.
constexpr int ST = 256;
constexpr int SWV = ST / WAVE;
constexpr int RC = 1024;         // requests of a chunk
constexpr int RPT = RC / ST;     // requests per thread

struct Req {       // a request's part of the step
  int64_t kept, add;
  int32_t held, need, lack, over;
  uint32_t status;
};

__device__ __forceinline__ Req request(const gsp_pages &p, const gsp_step &t, bool ring_ok, int r) {
  const int64_t len = p.counters[2 + r], keep = t.keep ? t.keep[r] : 0, add = t.add[r];
  Req q;
  q.held = p.counters[2 + (int64_t)p.requests + r];
  q.kept = keep < 0 ? 0 : len + keep;
  q.add = add;
  q.lack = q.over = 0;
  q.need = q.held;
  q.status = GSP_STEP_OK;
  if (!ring_ok || add < 0 || len < 0 || q.held < 0 || q.held > (int64_t)p.max_pages || q.kept > (int64_t)q.held * p.page) {
    q.status = GSP_STEP_BAD;
    q.kept = len;
    q.add = add < 0 ? 0 : add;
    return q;
  }
  const int64_t need = (q.kept + add + p.page - 1) / p.page;
  if (need > (int64_t)p.max_pages) {
    q.status = GSP_STEP_FULL;
    return q;
  }
  q.need = (int32_t)need;
  q.lack = max(q.need - q.held, 0);
  q.over = max(q.held - q.need, 0);
  return q;
}

struct StepShared {
  int64_t wsum[SWV];
  // the chunk's requests: first new token, kept length, pages held, first ring entry taken, status; first page given back
  int64_t tok[RC + 1];
  int64_t kept[RC], take[RC], give[RC + 1];
  int32_t held[RC], need[RC];
  uint32_t status[RC];
};

// Exclusive sums of v over the chunk (RPT consecutive requests a thread) on top of `carry`, which becomes the sum after it.
__device__ __forceinline__ void chunk_scan(const int64_t (&v)[RPT], int64_t (&out)[RPT], int64_t &carry, StepShared &sh) {
  int64_t s = 0;
  for (int k = 0; k < RPT; ++k) s += v[k];
  const int64_t inc = (int64_t)wave_incl_scan_u64((uint64_t)s);
  __syncthreads();
  if (lane_id() == WAVE - 1) sh.wsum[threadIdx.x >> 6] = inc;
  __syncthreads();
  int64_t base = carry + inc - s;
  for (int k = 0; k < (int)(threadIdx.x >> 6); ++k) base += sh.wsum[k];
  for (int k = 0; k < RPT; ++k) {
    out[k] = base;
    base += v[k];
  }
  for (int k = 0; k < SWV; ++k) carry += sh.wsum[k];
}

// The last i in [0, n) with first[i] <= x (first ascends, first[0] <= x).
__device__ __forceinline__ int find(const int64_t *first, int n, int64_t x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int m = (lo + hi) / 2;
    if (first[m] <= x) lo = m;
    else hi = m;
  }
  return lo;
}

// state: writes counters_out (one workgroup), else the step's outputs. Both, when the state goes to an array of its own.
template <bool OUTS, bool STATE>
__global__ __launch_bounds__(ST) void step_kernel(gsp_pages p, gsp_step t) {
  __shared__ StepShared sh;
  const int R = (int)p.requests, tid = threadIdx.x;
  const int64_t head = p.counters[0], free = p.counters[1];
  const bool ring_ok = head >= 0 && head < p.pool && free >= 0 && free <= p.pool;
  const int64_t gid = (int64_t)blockIdx.x * ST + tid, gsize = (int64_t)gridDim.x * ST;
  int64_t tokens = 0, lacking = 0, given = 0, taken = 0;  // sums before the chunk; taken: by the requests that were served
  for (int r0 = 0; r0 < R; r0 += RC) {
    Req q[RPT];
    int64_t v[RPT], tok[RPT], lack[RPT], give[RPT];
    const int64_t tok0 = tokens, give0 = given;
    for (int k = 0; k < RPT; ++k) {
      const int r = r0 + tid * RPT + k;
      q[k] = r < R ? request(p, t, ring_ok, r) : Req{};
      v[k] = q[k].add;
    }
    chunk_scan(v, tok, tokens, sh);
    for (int k = 0; k < RPT; ++k) v[k] = q[k].lack;
    chunk_scan(v, lack, lacking, sh);
    for (int k = 0; k < RPT; ++k) {
      if (q[k].status == GSP_STEP_OK &&
          ((q[k].lack > 0 && lack[k] + q[k].lack > free) || (q[k].add > 0 && tok[k] + q[k].add > (int64_t)t.max_tokens)))
        q[k].status = GSP_STEP_FULL;
      if (q[k].status != GSP_STEP_OK) {
        q[k].need = q[k].held;
        q[k].lack = q[k].over = 0;
      }
      v[k] = q[k].over;
    }
    chunk_scan(v, give, given, sh);
    int64_t most = 0;
    for (int k = 0; k < RPT; ++k)
      if (q[k].lack > 0) most = lack[k] + q[k].lack;
    taken = max(taken, (int64_t)wave_max_u64((uint64_t)most));  // (per wave; the state's thread joins the waves' below)
    __syncthreads();
    for (int k = 0; k < RPT; ++k) {
      const int i = tid * RPT + k, r = r0 + i;
      sh.tok[i] = tok[k];
      sh.kept[i] = q[k].kept;
      sh.take[i] = lack[k];
      sh.give[i] = give[k];
      sh.held[i] = q[k].held;
      sh.need[i] = q[k].need;
      sh.status[i] = q[k].status;
      if (r >= R) continue;
      if (OUTS && blockIdx.x == 0) {
        t.begin[r] = (int32_t)min(tok[k], (int64_t)INT32_MAX);
        t.status[r] = q[k].status;
        t.seq_len[r] = (int32_t)min(q[k].kept + (q[k].status == GSP_STEP_OK ? q[k].add : 0), (int64_t)INT32_MAX);
      }
      if (STATE && blockIdx.x == 0) {
        p.counters_out[2 + r] = (int32_t)q[k].kept;
        p.counters_out[2 + (int64_t)R + r] = q[k].need;
      }
    }
    if constexpr (OUTS) {
      const int n = min(RC, R - r0);
      __syncthreads();
      const int64_t end = min(tokens, (int64_t)t.max_tokens);
      for (int64_t i = tok0 + ((gid - tok0) % gsize + gsize) % gsize; i < end; i += gsize) {
        const int k = find(sh.tok, n, i);
        const int64_t at = sh.kept[k] + i - sh.tok[k];
        int64_t slot = -1;
        if (sh.status[k] == GSP_STEP_OK) {
          const int64_t pg = at / p.page, off = at - pg * p.page;
          int32_t *row = p.table + (int64_t)(r0 + k) * p.table_ld;
          int32_t id;
          if (pg < sh.held[k]) {
            id = row[pg];
          } else {
            id = p.ring[(head + sh.take[k] + pg - sh.held[k]) % p.pool];
            if (off == 0) row[pg] = id;
          }
          slot = (int64_t)id * p.page + off;
        }
        t.slot[i] = slot;
        if (t.pos) t.pos[i] = (int32_t)(t.depth ? sh.kept[k] + t.depth[i] : at);
        if (t.req) t.req[i] = r0 + k;
      }
      for (int64_t i = give0 + gid; i < given; i += gsize) {
        const int k = find(sh.give, n, i);
        p.ring[(head + free + i) % p.pool] = p.table[(int64_t)(r0 + k) * p.table_ld + sh.need[k] + i - sh.give[k]];
      }
    }
    __syncthreads();
  }
  if constexpr (OUTS) {
    for (int64_t i = min(tokens, (int64_t)t.max_tokens) + gid; i < (int64_t)t.max_tokens; i += gsize) {
      t.slot[i] = -1;
      if (t.pos) t.pos[i] = 0;
      if (t.req) t.req[i] = -1;
    }
    if (gid == 0) t.begin[R] = (int32_t)min(tokens, (int64_t)INT32_MAX);
  }
  if constexpr (STATE) {
    if (blockIdx.x == 0) {
      if (lane_id() == 0) sh.wsum[tid >> 6] = taken;
      __syncthreads();
      if (tid == 0) {
        for (int k = 0; k < SWV; ++k) taken = max(taken, sh.wsum[k]);
        p.counters_out[0] = (int32_t)(ring_ok ? (head + taken) % p.pool : head);
        p.counters_out[1] = (int32_t)(free - taken + given);
      }
    }
  }
}

// ---- the path -----------------------------------------------------------------------------------------------------------
// A thread copies one vector of one chunk of one cache along its request's path. Nodes ascend (node i >= i), so the slot
// that entry i goes to is the source of no later entry; the thread alone touches its column, in path order.
constexpr int PT = 256;

template <typename VEC>
__global__ __launch_bounds__(PT) void path_kernel(gsp_path a, int vecs) {
  const int r = blockIdx.y;
  const int64_t id = (int64_t)blockIdx.x * PT + threadIdx.x;  // (cache, chunk, vector)
  const int len = min(a.emit_len[r], (int)min(a.emit_ld, (int64_t)INT32_MAX));
  const int64_t anchor = a.anchor[r];
  if (id >= (int64_t)a.caches * a.chunks * vecs) return;
  const int64_t cc = id / vecs;
  const int64_t k = cc / a.chunks;
  char *base = (a.cache_ptrs ? (char *)a.cache_ptrs[k] : (char *)a.cache + k * a.cache_stride) + (cc % a.chunks) * a.chunk_stride +
               (id % vecs) * sizeof(VEC);
  const int64_t slots = (int64_t)a.pages * a.page;
  for (int i = 1; i < len; ++i) {
    const int64_t node = a.emit_nodes[r * a.emit_ld + i], to = anchor + i;
    if (node < 0 || node >= a.tokens || to < 0 || to >= a.tokens || node == to) continue;
    const int64_t s = a.slot[node], d = a.slot[to];
    if (s < 0 || s >= slots || d < 0 || d >= slots) continue;
    const VEC v = *(const VEC *)(base + s / a.page * a.page_stride + s % a.page * a.token_stride);
    *(VEC *)(base + d / a.page * a.page_stride + d % a.page * a.token_stride) = v;
  }
}

}  // namespace

hipError_t launch_pages(const gsp_pages &p, const gsp_step &t, hipStream_t s) {
  const int64_t wgs = ((int64_t)t.max_tokens + ST - 1) / ST;
  const dim3 grid((uint32_t)max((int64_t)1, min(wgs, (int64_t)1024)));
  if (p.counters_out != p.counters) {
    hipLaunchKernelGGL((step_kernel<true, true>), grid, dim3(ST), 0, s, p, t);
  } else {
    hipLaunchKernelGGL((step_kernel<true, false>), grid, dim3(ST), 0, s, p, t);
    hipLaunchKernelGGL((step_kernel<false, true>), dim3(1), dim3(ST), 0, s, p, t);
  }
  return hipGetLastError();
}

hipError_t launch_path(const gsp_path &p, hipStream_t s) {
  auto go = [&](auto v) {
    using V = decltype(v);
    const int vecs = (int)(p.chunk_bytes / sizeof(V));
    const int64_t ids = (int64_t)p.caches * p.chunks * vecs;
    for (uint32_t r0 = 0; r0 < p.requests; r0 += 65535) {
      gsp_path a = p;
      a.requests = min(p.requests - r0, 65535u);
      a.anchor += r0;
      a.emit_len += r0;
      a.emit_nodes += r0 * p.emit_ld;
      hipLaunchKernelGGL((path_kernel<V>), dim3((uint32_t)((ids + PT - 1) / PT), a.requests), dim3(PT), 0, s, a, vecs);
    }
  };
  // the widest vector that every address is a multiple of
  const uint64_t all = (uint64_t)p.chunk_bytes | (uint64_t)p.page_stride | (uint64_t)p.token_stride | (uint64_t)p.chunk_stride |
                       (p.cache_ptrs ? (uint64_t)p.align : (uint64_t)p.cache | (uint64_t)p.cache_stride);
  if (all % 16 == 0) go(uint4{});
  else if (all % 4 == 0) go(uint32_t{});
  else if (all % 2 == 0) go(uint16_t{});
  else go(uint8_t{});
  return hipGetLastError();
}

}  // namespace gse
