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
// Every workgroup (of ST threads) forms the sums itself (16 bytes a request, from cache), ST requests at a time, one a thread,
// so no workgroup waits for another; then it takes its tiles of ST of the chunk's tokens and its share of the pages given
// back. The state is read from counters and written to counters_out by one workgroup: when they are the same array, by a
// second launch. Bound by the chain of state, scan, search and page reads: 3.9 us for a request, 6.1 for 512; 1024 requests with
// a map of 2^20 entries (17 MB written) 10.9 us.

struct Req {       // a request's part of the step
  int64_t kept, add;
  int32_t held, need, lack, over;
  uint32_t status;
};

__device__ __forceinline__ Req request(const gsp_pages &p, bool ring_ok, int64_t len, int64_t held, int64_t keep, int64_t add) {
  Req q;
  q.held = (int32_t)held;
  q.kept = keep < 0 ? 0 : len + keep;
  q.add = add;
  q.lack = q.over = 0;
  q.need = q.held;
  q.status = GSP_STEP_OK;
  if (!ring_ok || add < 0 || len < 0 || held < 0 || held > (int64_t)p.max_pages || q.kept > held * p.page) {
    q.status = GSP_STEP_BAD;
    q.kept = len;
    q.add = add < 0 ? 0 : add;
    return q;
  }
  const uint32_t total = (uint32_t)(q.kept + add);  // (max_pages * page < 2^31: both are below 2^31)
  const uint32_t need = total / p.page + (total % p.page != 0);
  if (need > p.max_pages) {
    q.status = GSP_STEP_FULL;
    return q;
  }
  q.need = (int32_t)need;
  q.lack = max(q.need - q.held, 0);
  q.over = max(q.held - q.need, 0);
  return q;
}

constexpr uint32_t UNSERVED = 0x80000000u;

template <int ST>
struct StepShared {
  // the chunk's requests: first new token (from the chunk's first); that, the kept length (with UNSERVED), the pages held and
  // the ring index of the first page taken; the first page given back (from the chunk's first) and the pages needed
  uint32_t tok[ST];
  uint4 info[ST];
  uint32_t give[ST], need[ST];
  int64_t wave[3][ST / WAVE];
};

// The last i in [0, n) with first[i] <= x (first ascends, first[0] <= x).
__device__ __forceinline__ int find(const uint32_t *first, int n, uint32_t x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int m = (lo + hi) / 2;
    if (first[m] <= x) lo = m;
    else hi = m;
  }
  return lo;
}

// The exclusive prefix of the thread's s over the workgroup, on top of carry, which becomes the sum after it; inc: the
// inclusive prefix in the wave, wave: the waves' sums (scanned by every wave; added up one after the other, the step of 1024
// requests took 13.2 us).
template <int N>
__device__ __forceinline__ int64_t block_prefix(int64_t s, int64_t inc, int64_t &carry, const int64_t (&wave)[N]) {
  const int lane = lane_id(), wv = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint64_t to = wave_incl_scan_u64(lane < N ? (uint64_t)wave[lane] : 0ull);
  const int64_t base = carry + inc - s + (wv > 0 ? (int64_t)shfl_u64(to, wv - 1) : 0);
  carry += (int64_t)lane63(to);
  return base;
}

// OUTS: writes the step's outputs. STATE: its first workgroup writes counters_out.
template <int ST, bool OUTS, bool STATE>
__global__ __launch_bounds__(ST) void step_kernel(gsp_pages p, gsp_step t) {
  __shared__ StepShared<ST> sh;
  const int R = (int)p.requests, tid = threadIdx.x, wv = tid >> 6, lane = lane_id();
  const bool first = blockIdx.x == 0;
  const int64_t head = p.counters[0], free = p.counters[1], pool = p.pool;
  const bool ring_ok = head >= 0 && head < pool && free >= 0 && free <= pool;
  int64_t tokens = 0, lacking = 0, given = 0, taken = 0;  // sums before the chunk; taken: by the requests that were served
  for (int r0 = 0; r0 < R; r0 += ST) {
    if (r0) __syncthreads();
    const int n = min(ST, R - r0), r = r0 + tid;
    Req q = {};
    bool ends = false;
    if (tid < n) {
      int32_t keep = t.keep ? t.keep[r] : 0;
      if (keep > 0 && t.laid && t.laid[r] != GSP_STEP_OK) keep = 0;  // (they were written nowhere)
      ends = keep < 0;
      q = request(p, ring_ok, p.counters[2 + r], p.counters[2 + (int64_t)R + r], keep, t.add[r]);
    }
    const int64_t it = (int64_t)wave_incl_scan_u64((uint64_t)q.add), il = (int64_t)wave_incl_scan_u64((uint64_t)q.lack);
    if (lane == WAVE - 1) {
      sh.wave[0][wv] = it;
      sh.wave[1][wv] = il;
    }
    __syncthreads();
    const int64_t tok0 = tokens, give0 = given;
    const int64_t tok = block_prefix(q.add, it, tokens, sh.wave[0]), take = block_prefix(q.lack, il, lacking, sh.wave[1]);
    if (q.status == GSP_STEP_OK &&
        ((q.lack > 0 && take + q.lack > free) || (q.add > 0 && tok + q.add > (int64_t)t.max_tokens)))
      q.status = GSP_STEP_FULL;
    if (q.status != GSP_STEP_OK) {  // (a request that ends gives its pages back though what starts in its place does not fit)
      q.need = q.status == GSP_STEP_FULL && ends ? 0 : q.held;
      q.lack = 0;
      q.over = q.held - q.need;
    }
    if (q.lack > 0) taken = take + q.lack;
    const int64_t ig = (int64_t)wave_incl_scan_u64((uint64_t)q.over);
    if (lane == WAVE - 1) sh.wave[2][wv] = ig;
    __syncthreads();
    const int64_t give = block_prefix(q.over, ig, given, sh.wave[2]);
    if (tid < n) {
      const bool ok = q.status == GSP_STEP_OK;
      if constexpr (OUTS) {
        const int64_t at = head + take;
        sh.tok[tid] = (uint32_t)min(tok - tok0, (int64_t)UINT32_MAX);
        sh.info[tid] = uint4{(uint32_t)min(tok - tok0, (int64_t)UINT32_MAX), (uint32_t)q.kept | (ok ? 0u : UNSERVED),
                             (uint32_t)q.held, (uint32_t)(at >= pool ? at - pool : at)};
        sh.give[tid] = (uint32_t)(give - give0);
        sh.need[tid] = (uint32_t)q.need;
        if (first) {
          t.begin[r] = (int32_t)min(tok, (int64_t)INT32_MAX);
          t.status[r] = q.status;
          t.seq_len[r] = (int32_t)(q.kept + (ok ? q.add : 0));
        }
      }
      if (STATE && first) {
        p.counters_out[2 + r] = (int32_t)q.kept;
        p.counters_out[2 + (int64_t)R + r] = q.need;
      }
    }
    if constexpr (OUTS) {
      __syncthreads();
      const int64_t end = min(tokens, (int64_t)t.max_tokens);
      int64_t tile = tok0 / ST;
      tile += (blockIdx.x + (int64_t)gridDim.x - tile % gridDim.x) % gridDim.x;
      for (; tile * ST < end; tile += gridDim.x) {
        const int64_t i = tile * ST + tid;
        if (i < tok0 || i >= end) continue;
        const uint32_t rel = (uint32_t)(i - tok0);
        const int m = find(sh.tok, n, rel);
        const uint4 f = sh.info[m];
        const uint32_t kept = f.y & ~UNSERVED, at = kept + (rel - f.x);
        int64_t slot = -1;
        if (!(f.y & UNSERVED)) {
          const uint32_t pg = at / p.page, off = at - pg * p.page;
          int32_t *row = p.table + (int64_t)(r0 + m) * p.table_ld;
          int32_t id;
          if (pg < f.z) {
            id = row[pg];
          } else {
            uint32_t g = f.w + (pg - f.z);
            if (g >= p.pool) g -= p.pool;
            id = p.ring[g];
            if (off == 0) row[pg] = id;
          }
          slot = (int64_t)id * p.page + off;
        }
        t.slot[i] = slot;
        if (t.pos) t.pos[i] = (int32_t)(t.depth ? kept + (uint32_t)t.depth[i] : at);
        if (t.req) t.req[i] = r0 + m;
      }
      for (int64_t i = (int64_t)blockIdx.x * ST + tid; i < given - give0; i += (int64_t)gridDim.x * ST) {
        const int m = find(sh.give, n, (uint32_t)i);
        p.ring[(head + free + give0 + i) % pool] = p.table[(int64_t)(r0 + m) * p.table_ld + sh.need[m] + (i - sh.give[m])];
      }
    }
  }
  if constexpr (OUTS) {
    const int64_t end = min(tokens, (int64_t)t.max_tokens);
    for (int64_t i = end + (int64_t)blockIdx.x * ST + tid; i < (int64_t)t.max_tokens; i += (int64_t)gridDim.x * ST) {
      t.slot[i] = -1;
      if (t.pos) t.pos[i] = 0;
      if (t.req) t.req[i] = -1;
    }
    if (first && tid == 0) t.begin[R] = (int32_t)min(tokens, (int64_t)INT32_MAX);
  }
  if constexpr (STATE) {
    if (first) {
      const int64_t most = (int64_t)wave_max_u64((uint64_t)taken);
      __syncthreads();
      if (lane == 0) sh.wave[0][wv] = most;
      __syncthreads();
      if (tid == 0) {
        for (int k = 0; k < ST / WAVE; ++k) taken = max(taken, sh.wave[0][k]);
        p.counters_out[0] = (int32_t)(ring_ok ? (head + taken) % pool : head);
        p.counters_out[1] = (int32_t)(free - taken + given);
      }
    }
  }
}

// ---- the path -----------------------------------------------------------------------------------------------------------
// A thread moves the vectors of its columns (a column: one place in one chunk of one cache) of every entry of its request's
// path. The workgroup's first wave finds 64 entries' slots at once (a lane an entry: three dependent reads in all, whatever
// the path's length) and leaves their offsets in LDS; every thread then loads up to four entries' vectors before it stores
// them. Nodes ascend along a path, so entry i's target, i places after the anchor, is the source of no later entry, and loads
// ahead of the stores read what was there before the call. A column belongs to one thread: nothing is shared but the offsets.
// Bound by latency, then by memory: 64 paths of up to four entries over 64 caches (17.6 MB read and written) 7.1 us with an
// entry at a time and every wave finding the slots, 5.1 so (3.4 TB/s); a group of four filled up with its last entry, stored
// again, took 19.6.
constexpr int PT = 256;
constexpr int64_t PATH_WGS = 2048;  // workgroups of a launch to aim for: a thread then has a column or a few (64 paths over 64
                                    // caches of 2 KB rows: 512, 1024, 2048, 4096 workgroups 6.9, 5.6, 5.1, 5.1 us)

struct PathShared {
  int64_t src[WAVE], dst[WAVE];  // byte offsets of the entries that move
  int n;
};

template <typename VEC>
__global__ __launch_bounds__(PT) void path_kernel(gsp_path a, uint32_t vecs) {
  __shared__ PathShared sh;
  const int r = blockIdx.y, tid = threadIdx.x, lane = lane_id();
  const int64_t len = min((int64_t)a.emit_len[r], a.emit_ld), anchor = a.anchor[r];
  const uint64_t slots = (uint64_t)a.pages * a.page;  // (below 2^32)
  auto offset = [&](uint32_t s) {
    const uint32_t pg = s / a.page;
    return (int64_t)pg * a.page_stride + (int64_t)(s - pg * a.page) * a.token_stride;
  };
  const uint32_t columns = a.caches * a.chunks * vecs;
  for (int64_t i0 = 1; i0 < a.emit_ld; i0 += WAVE) {
    if (i0 > 1) __syncthreads();
    if (tid < WAVE) {
      const int64_t i = i0 + lane, to = anchor + i;
      const int64_t node = i < a.emit_ld ? a.emit_nodes[r * a.emit_ld + i] : -1;  // (read ahead of the length)
      bool moves = i < len && node >= 0 && node < a.tokens && anchor >= 0 && to < a.tokens && node != to;
      uint64_t s = 0, d = 0;
      if (moves) {
        s = (uint64_t)a.slot[node];
        d = (uint64_t)a.slot[to];
        moves = s < slots && d < slots;  // (negative ones are past them)
      }
      const uint64_t m = ballot64(moves);
      const int n = (int)__popcll(m);
      if (moves) {
        const int64_t so = offset((uint32_t)s), to_ = offset((uint32_t)d);
        const int k = (int)lanes_below(m);
        sh.src[k] = so;
        sh.dst[k] = to_;
      }
      if (lane == 0) sh.n = n;
    }
    __syncthreads();
    const int n = sh.n;
    if (n > 0) {
      for (uint32_t id = blockIdx.x * PT + tid; id < columns; id += gridDim.x * PT) {
        const uint32_t cc = id / vecs, k = cc / a.chunks;
        char *base = a.cache_ptrs ? (char *)a.cache_ptrs[k] : (char *)a.cache + k * a.cache_stride;
        base += (int64_t)(cc - k * a.chunks) * a.chunk_stride + (int64_t)(id - cc * vecs) * sizeof(VEC);
        int e = 0;
        for (; e + 4 <= n; e += 4) {
          const VEC v0 = *(const VEC *)(base + sh.src[e]), v1 = *(const VEC *)(base + sh.src[e + 1]);
          const VEC v2 = *(const VEC *)(base + sh.src[e + 2]), v3 = *(const VEC *)(base + sh.src[e + 3]);
          *(VEC *)(base + sh.dst[e]) = v0;
          *(VEC *)(base + sh.dst[e + 1]) = v1;
          *(VEC *)(base + sh.dst[e + 2]) = v2;
          *(VEC *)(base + sh.dst[e + 3]) = v3;
        }
        for (; e + 2 <= n; e += 2) {
          const VEC v0 = *(const VEC *)(base + sh.src[e]), v1 = *(const VEC *)(base + sh.src[e + 1]);
          *(VEC *)(base + sh.dst[e]) = v0;
          *(VEC *)(base + sh.dst[e + 1]) = v1;
        }
        if (e < n) {
          const VEC v0 = *(const VEC *)(base + sh.src[e]);
          *(VEC *)(base + sh.dst[e]) = v0;
        }
      }
    }
    if (i0 + WAVE >= len) break;
  }
}

}  // namespace

hipError_t launch_pages(const gsp_pages &p, const gsp_step &t, hipStream_t s) {
  // A thread a request, up to 1024 (96 requests: workgroups of 256 with a request a thread 4.5 us, with four 5.8; 512: 6.2 with
  // 512 threads, 6.8 with 256 of four); 2^18 threads over the tokens: every workgroup forms the sums anew (1024 requests,
  // 2^20 tokens: 2^17, 2^18, 2^19 threads 12.2, 10.9, 13.1 us). In place, the second launch: a request 3.9 -> 6.1 us, 512 6.2 ->
  // 8.6, 1024 with the map 10.8 -> 15.0.
  constexpr int64_t threads = 1 << 18;
  auto go = [&](auto st) {
    constexpr int ST = decltype(st)::value;
    const int64_t tiles = ((int64_t)t.max_tokens + ST - 1) / ST;
    const dim3 grid((uint32_t)max((int64_t)1, min(tiles, threads / ST)));
    if (p.counters_out != p.counters) {
      hipLaunchKernelGGL((step_kernel<ST, true, true>), grid, dim3(ST), 0, s, p, t);
    } else {
      hipLaunchKernelGGL((step_kernel<ST, true, false>), grid, dim3(ST), 0, s, p, t);
      hipLaunchKernelGGL((step_kernel<ST, false, true>), dim3(1), dim3(ST), 0, s, p, t);
    }
  };
  if (p.requests <= 256) go(std::integral_constant<int, 256>{});
  else if (p.requests <= 512) go(std::integral_constant<int, 512>{});
  else go(std::integral_constant<int, 1024>{});
  return hipGetLastError();
}

hipError_t launch_path(const gsp_path &p, hipStream_t s) {
  auto go = [&](auto v) {
    using V = decltype(v);
    const uint32_t vecs = (uint32_t)(p.chunk_bytes / sizeof(V));
    const int64_t ids = (int64_t)p.caches * p.chunks * vecs;  // (at most 2^30)
    const int64_t all = (ids + PT - 1) / PT, wgs = min(all, max((int64_t)1, PATH_WGS / p.requests));
    for (uint32_t r0 = 0; r0 < p.requests; r0 += 65535) {
      gsp_path a = p;
      a.requests = min(p.requests - r0, 65535u);
      a.anchor += r0;
      a.emit_len += r0;
      a.emit_nodes += r0 * p.emit_ld;
      hipLaunchKernelGGL((path_kernel<V>), dim3((uint32_t)wgs, a.requests), dim3(PT), 0, s, a, vecs);
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
