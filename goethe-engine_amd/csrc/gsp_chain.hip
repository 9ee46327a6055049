// Drafted chains against the target's probability rows (gsp_verify_chains): the accepted length of every request and the
// token drawn after it.
//
// With p_i the target's row after i drafts and q_i the row that draft x_i was drawn from, draft i is accepted iff
// q_i(x_i) > 0 and coin_i q_i(x_i) < p_i(x_i): with probability min(1, p / q). At the first draft a that is not, the token
// comes from max(p_a - q_a, 0), which makes its law p_a again; after the last one from p_n. The tests read two values per
// draft, so what has to be read is one row of p per request, and one of q where a draft was rejected.
//
// A request's row is cut into segments that a wave sums alone, 16 bytes a lane and load, in fp64 (a token is an index: sums in
// fp32 would move it); the last workgroup in, by a ticket, finds the segment, then the token that u times the sum falls
// into. One launch, whatever the chains' lengths. Bound by memory in large calls: 512 chains over 262144 bf16 tokens read
// 390 MB in 71 us, 5.5 TB/s (a large copy: 5.1), 6.9 VALU instructions a token; a call of few rows is the chain of
// dependent reads offsets, drafts, their weights, the row, the sums, the token's segment: 6.1 us for one chain over 128256
// fp32 tokens. One workgroup a request and two passes took 2260 and 275 us; a workgroup a slice of 32 KB (8192 of them, each
// through the first three reads and a ticket) 173 us.
#include "gse_dev.h"
#include "gsp_int.h"

namespace gse {

namespace {

constexpr int CT = 256;          // threads of a workgroup
constexpr int CW = CT / WAVE;
// Workgroups of a request, at most: each ends with an atomic on the request's ticket. One chain over 128256 fp32 tokens with 8,
// 16, 32, 48, 64, 128: 7.3, 6.1, 6.2, 6.1, 6.6, 6.7 us; 16 chains over 151936 fp64 tokens 19.4, 14.9, 13.2, 10.2, 11.1, 11.1.
constexpr int WGS_MAX = 48;

template <int T>
constexpr int SIZE = T == GSP_F64 ? 8 : T == GSP_F32 ? 4 : 2;
template <int T>
__device__ __forceinline__ const char *row_of(const void *base, int64_t ld, int64_t row) {
  return (const char *)base + row * ld * SIZE<T>;
}
// One value of a row of type T as fp64 (exact for every type).
template <int T>
__device__ __forceinline__ double value(const char *row, int64_t t) {
  if constexpr (T == GSP_F64) return ((const double *)row)[t];
  else if constexpr (T == GSP_F32) return (double)((const float *)row)[t];
  else if constexpr (T == GSP_BF16) return (double)bf16_to_f32(((const uint16_t *)row)[t]);
  else return (double)((const _Float16 *)row)[t];
}

// N consecutive values of a row of type T, as loaded (rows start at any element: the loads need no more alignment than one).
// NT: read past the caches' keeping.
template <int T, int N>
struct Raw {
  static constexpr int W = SIZE<T> * N / 4;
  typedef uint32_t Q __attribute__((ext_vector_type(W), aligned(2)));
  uint32_t w[W];
  template <bool NT>
  __device__ __forceinline__ void load(const char *row, int64_t t) {
    const Q *at = (const Q *)(row + t * SIZE<T>);
    Q q;
    if constexpr (NT) q = __builtin_nontemporal_load(at);
    else q = *at;
#pragma unroll
    for (int i = 0; i < W; ++i) w[i] = q[i];
  }
  __device__ __forceinline__ double get(int i) const {
    if constexpr (T == GSP_F64) return __hiloint2double((int)w[2 * i + 1], (int)w[2 * i]);
    else if constexpr (T == GSP_F32) return (double)__uint_as_float(w[i]);
    else if constexpr (T == GSP_BF16) return (double)__uint_as_float(i & 1 ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16);
    else return (double)__builtin_bit_cast(_Float16, (uint16_t)(i & 1 ? w[i / 2] >> 16 : w[i / 2]));
  }
};

struct ChainEnd {
  int a;         // accepted drafts (-1: begin is out of order)
  int x;         // the draft rejected after them, -1: the chain ended
  int64_t row;   // the target row the token is drawn from; the rejected draft's row of q is row - request
};

// The chain of request r, by one wave (every lane gets the answer): 64 drafts at a time. emit: also writes the accepted
// drafts and the padding after the last token's place.
template <int PT, int QT>
__device__ __forceinline__ ChainEnd chain_end(const gsp_chains &c, int r, bool emit) {
  const int lane = lane_id(), V = (int)c.vocab;
  const int b0 = __builtin_amdgcn_readfirstlane(c.begin[r]), b1 = __builtin_amdgcn_readfirstlane(c.begin[r + 1]);
  ChainEnd e{-1, -1, 0};
  const bool good = b0 >= 0 && b1 >= b0 && b1 <= (int)c.drafts && b1 - b0 <= (int)c.max_drafts;
  const int n = good ? b1 - b0 : 0;
  e.a = good ? n : -1;
  for (int i0 = 0; i0 < n; i0 += WAVE) {
    const int i = i0 + lane;
    const int x = i < n ? c.token[b0 + i] : -1;
    const bool in = x >= 0 && x < V;
    double px = 0.0;
    bool took = false;
    if (in) {
      px = value<PT>(row_of<PT>(c.target, c.target_ld, (int64_t)b0 + r + i), x);
      const double qx = QT < 0 ? 1.0 : value<QT>(row_of<QT>(c.draft, c.draft_ld, (int64_t)b0 + i), x);
      took = qx > 0.0 && c.coin[b0 + i] * qx < px;
    }
    const uint64_t miss = ballot64(!took);
    const int f = miss ? (int)__builtin_ctzll(miss) : WAVE;
    if (emit && lane < f) {
      c.emit_tokens[r * c.emit_ld + i] = x;
      if (c.emit_probs) c.emit_probs[r * c.emit_ld + i] = (float)px;
    }
    if (f < WAVE) {
      e.a = i0 + f;
      const int xf = __builtin_amdgcn_readlane(x, f);
      e.x = xf < V ? xf : -1;  // (-1: past the chain's end, or a pad)
      break;
    }
  }
  if (e.a > n) e.a = n;
  if (e.x < 0) e.x = -1;
  e.row = (int64_t)b0 + r + max(e.a, 0);
  if (emit)
    for (int i = e.a + 1 + lane; i <= (int)c.max_drafts; i += WAVE) {
      c.emit_tokens[r * c.emit_ld + i] = -1;
      if (c.emit_probs) c.emit_probs[r * c.emit_ld + i] = 0.0f;
    }
  return e;
}

// The distribution that a request's token is drawn from: weight(t) = max(p(t) - q(t), 0), q null: max(p(t), 0), and x's
// weight 0. The kernel sums v + |v| = 2 max(v, 0), v = p - q, which is exact, one add, and unlike a maximum keeps what is not
// finite: a NaN or an infinity anywhere in the rows makes the sum NaN or infinite. Every sum and threshold is so doubled.
struct ChainRow {
  const char *p, *q;
  int x;
};

template <int PT, int QT, int VEC, bool HQ>
struct Weights {
  static constexpr int Q = HQ ? QT : GSP_BF16;
  Raw<PT, VEC> p;
  Raw<Q, HQ ? VEC : 2> q;
  template <bool NT>
  __device__ __forceinline__ void load(const ChainRow &w, int64_t t) {
    p.template load<NT>(w.p, t);
    if constexpr (HQ) q.template load<NT>(w.q, t);
  }
  __device__ __forceinline__ double get(int i) const {
    double v = p.get(i);
    if constexpr (HQ) v -= q.get(i);
    return v + fabs(v);
  }
};

template <int PT, int QT, bool HQ>
__device__ __forceinline__ double weight(const ChainRow &w, int t) {
  double v = value<PT>(w.p, t);
  if constexpr (HQ) v -= value<QT>(w.q, t);
  return t == w.x ? 0.0 : v + fabs(v);
}

// A row's vectors of VEC tokens go to segments of S * 64: vector k * 64 + lane of a segment is a lane's k-th. The tokens past
// the row's last whole vector (fewer than VEC) go with the last segment, one a lane.
struct ChainArgs {
  gsp_chains c;
  int r0;          // first request of the launch
  int nseg;        // segments of a row
  double *sum;     // [requests of the launch][nseg]
  // The ticket of request k of the launch at k * tstride, zero between calls. A cache line apart where there is room: side by
  // side, the atomics of all requests queue for one line (16 chains of 64 workgroups 20.6 us, apart 12.5).
  uint32_t *tick;
  int tstride;
};

template <int PT, int QT, int VEC, bool HQ>
__device__ __forceinline__ double tail_weight(const ChainRow &w, int V) {
  const int t = V / VEC * VEC + lane_id();
  return t < V ? weight<PT, QT, HQ>(w, t) : 0.0;
}

// The sum of a segment (last: with the row's tail), by one wave; every lane gets it.
template <int PT, int QT, int VEC, int S, bool HQ, bool NT>
__device__ __forceinline__ double segment_sum(const ChainRow &w, int seg, bool last, int V) {
  const int nv = V / VEC, i0 = seg * (S * WAVE), lane = lane_id();
  double a = 0.0;
  if (i0 + S * WAVE <= nv && (w.x < i0 * VEC || w.x >= (i0 + S * WAVE) * VEC)) {  // whole, and w.x not in it
    Weights<PT, QT, VEC, HQ> x[S];
#pragma unroll
    for (int k = 0; k < S; ++k) x[k].template load<NT>(w, (int64_t)(i0 + k * WAVE + lane) * VEC);
    // Every load before the first sum (the compiler had each fp64 pair waited for: 256 fp64 chains over 128256 tokens 104 -> 90
    // us, 64 fp32 ones 14.9 -> 14.5).
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int k = 0; k < S; ++k) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) a += x[k].get(e);
    }
  } else {
    for (int i = i0 + lane; i < min(i0 + S * WAVE, nv); i += WAVE) {
      Weights<PT, QT, VEC, HQ> x;
      x.template load<NT>(w, (int64_t)i * VEC);
#pragma unroll
      for (int e = 0; e < VEC; ++e) a += i * VEC + e == w.x ? 0.0 : x.get(e);
    }
  }
  if (last) a += tail_weight<PT, QT, VEC, HQ>(w, V);
  return wave_sum_f64(a);
}

// The first token of a segment (last: and of the row's tail) with a positive weight whose prefix, from `before` on, reaches
// thr (found); the last token with a positive weight when none does, -1 when there is none. before becomes the prefix after
// the segment where none does. By one wave; every lane gets it.
template <int PT, int QT, int VEC, int S, bool HQ>
__device__ __forceinline__ int segment_search(const ChainRow &w, int seg, bool last, int V, double &before, double thr,
                                              bool &found) {
  const int nv = V / VEC, i0 = seg * (S * WAVE), lane = lane_id();
  int lst = -1;
  constexpr int H = S < 4 ? S : 4;  // vectors a lane loads at once
  Weights<PT, QT, VEC, HQ> x[H];
#pragma unroll
  for (int k = 0; k < S; ++k) {
    if (k % H == 0 && nv > 0) {  // (past the last vector: that one again, not counted)
#pragma unroll
      for (int j = 0; j < H; ++j) x[j].template load<false>(w, (int64_t)min(i0 + (k + j) * WAVE + lane, nv - 1) * VEC);
      __builtin_amdgcn_sched_barrier(0);
    }
    const int i = i0 + k * WAVE + lane;
    double b[VEC], a = 0.0;
#pragma unroll
    for (int e = 0; e < VEC; ++e) a += b[e] = i < nv && i * VEC + e != w.x ? x[k % H].get(e) : 0.0;
    const double inc = before + wave_incl_scan_f64(a), up = shfl_up_f64(inc, 1);
    // this lane's tokens: the first that reaches thr, the last with a weight
    double at = lane > 0 ? up : before;
    int hit = -1, pos = -1;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      at += b[e];
      if (b[e] > 0.0) {
        pos = i * VEC + e;
        if (hit < 0 && !(at < thr)) hit = pos;
      }
    }
    const uint64_t pm = ballot64(pos >= 0);
    // the first lane whose vector reaches thr by the scan: its own sum, in another order, may stay below
    const uint64_t hm = ballot64(pos >= 0 && !(inc < thr));
    found = hm != 0;
    if (found) return __builtin_amdgcn_readlane(hit >= 0 ? hit : pos, (int)__builtin_ctzll(hm));
    if (pm) lst = __builtin_amdgcn_readlane(pos, 63 - (int)__builtin_clzll(pm));
    before = shfl_f64(inc, WAVE - 1);
  }
  if (last) {
    const int t = V / VEC * VEC + lane;
    const double b = tail_weight<PT, QT, VEC, HQ>(w, V);
    const double inc = before + wave_incl_scan_f64(b);
    const uint64_t pm = ballot64(b > 0.0), hm = ballot64(b > 0.0 && !(inc < thr));
    found = hm != 0;
    if (found) return __builtin_amdgcn_readlane(t, (int)__builtin_ctzll(hm));
    if (pm) lst = __builtin_amdgcn_readlane(t, 63 - (int)__builtin_clzll(pm));
    before = shfl_f64(inc, WAVE - 1);
  }
  return lst;
}

// The token drawn from a row whose segments are summed, by one wave; -1: an error.
template <int PT, int QT, int VEC, int S, bool HQ>
__device__ __forceinline__ int chain_draw(const ChainRow &w, const double *sum, int nseg, int V, double u, double &total) {
  constexpr int NB = 8;  // 64 sums each, loaded at once: a row of up to 512 segments waits for one round of loads
  const int lane = lane_id();
  double x[NB];
  auto block = [&](int b0) {
#pragma unroll
    for (int k = 0; k < NB; ++k) x[k] = b0 + k * WAVE + lane < nseg ? ld_ag(&sum[b0 + k * WAVE + lane]) : 0.0;
  };
  total = 0.0;
  for (int b0 = 0; b0 < nseg; b0 += NB * WAVE) {
    block(b0);
    double t = 0.0;
#pragma unroll
    for (int k = 0; k < NB; ++k) t += x[k];
    total += wave_sum_f64(t);
  }
  if (!(total > 0.0 && total < INFINITY)) return -1;
  const double thr = u * total;
  double before = 0.0, lb = 0.0;
  int lst = -1;  // the segment that the draw falls into: the first that reaches thr, else the last with a weight
  bool hit = false;
  for (int b0 = 0; b0 < nseg && !hit; b0 += NB * WAVE) {
    if (nseg > NB * WAVE) block(b0);
#pragma unroll
    for (int k = 0; k < NB; ++k) {
      if (hit || b0 + k * WAVE >= nseg) continue;
      const double inc = before + wave_incl_scan_f64(x[k]);
      const uint64_t pos = ballot64(x[k] > 0.0), hm = ballot64(x[k] > 0.0 && !(inc < thr));
      hit = hm != 0;
      if (pos) {
        const int l = hit ? (int)__builtin_ctzll(hm) : 63 - (int)__builtin_clzll(pos);
        lst = b0 + k * WAVE + l;
        lb = l > 0 ? shfl_f64(inc, l - 1) : before;
      }
      before = shfl_f64(inc, WAVE - 1);
    }
  }
  bool found = false;
  return segment_search<PT, QT, VEC, S, HQ>(w, lst, lst == nseg - 1, V, lb, thr, found);
}

// The same from p alone, nothing summed yet: where p is nowhere above q. One wave over the row twice (a row of
// 128256 fp32 tokens 206 us, of 262144 bf16 112, of 151936 fp64 339; with something left 6.2, 6.6, 7.4): with rows that sum to
// one only rounding (of p and q to their types, of the product with the coin) leads here.
template <int PT, int QT, int VEC, int S>
__device__ __noinline__ int chain_draw_again(const char *p, int nseg, int V, double u) {
  const ChainRow w{p, nullptr, -1};
  double total = 0.0, before = 0.0;
#pragma unroll 1
  for (int i = 0; i < nseg; ++i) total += segment_sum<PT, QT, VEC, S, false, false>(w, i, i == nseg - 1, V);
  if (!(total > 0.0 && total < INFINITY)) return -1;
  int lst = -1;
  bool found = false;
#pragma unroll 1
  for (int i = 0; i < nseg && !found; ++i) {
    const int j = segment_search<PT, QT, VEC, S, false>(w, i, i == nseg - 1, V, before, u * total, found);
    if (j >= 0) lst = j;
  }
  return lst;
}

// gridDim.x workgroups a request. Every wave finds the chain's end by itself (its drafts' values are cached after the first),
// then sums its share of the row's segments; the last workgroup's first wave (by a ticket) draws the token. No barrier but
// the ticket's, nothing in LDS but its answer.
template <int PT, int QT, int S, bool NT>
__global__ __launch_bounds__(CT) __attribute__((amdgpu_waves_per_eu(4, 8))) void chain_kernel(ChainArgs a) {
  constexpr int QS = QT < 0 ? 0 : SIZE<QT < 0 ? 0 : QT>;
  constexpr int VEC = 16 / (QS > SIZE<PT> ? QS : SIZE<PT>);
  __shared__ uint32_t ticket;
  const gsp_chains &c = a.c;
  const int k = blockIdx.y, r = a.r0 + k, tid = threadIdx.x, lane = lane_id(), V = (int)c.vocab;
  const int wv = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * CW + (tid >> 6)));  // the wave among the request's
  const int waves = (int)gridDim.x * CW;
  const ChainEnd e = chain_end<PT, QT>(c, r, wv == 0);
  ChainRow w{row_of<PT>(c.target, c.target_ld, e.row), nullptr, -1};
  if (e.x >= 0) {
    if constexpr (QT >= 0) w.q = row_of<QT>(c.draft, c.draft_ld, e.row - r);
    else w.x = e.x;
  }
  double *sum = a.sum + (int64_t)k * a.nseg;
  auto sums = [&](auto hq) {
    for (int i = wv; i < a.nseg; i += waves) {
      const double t = segment_sum<PT, QT, VEC, S, decltype(hq)::value, NT>(w, i, i == a.nseg - 1, V);
      if (lane == 0) st_ag(&sum[i], t);
    }
  };
  if (e.a >= 0) {
    if constexpr (QT >= 0) {
      if (w.q) sums(std::true_type{});
      else sums(std::false_type{});
    } else {
      sums(std::false_type{});
    }
  }
  store_wait();
  __syncthreads();
  if (tid == 0) ticket = ticket_add(&a.tick[k * a.tstride]);
  __syncthreads();
  if (ticket != gridDim.x - 1 || tid >= WAVE) return;
  int j = -1;
  if (e.a >= 0) {
    const double u = c.u[c.u_rows ? e.row : (int64_t)r];
    double total = 0.0;
    if constexpr (QT >= 0) {
      if (w.q) j = chain_draw<PT, QT, VEC, S, true>(w, sum, a.nseg, V, u, total);
      else j = chain_draw<PT, QT, VEC, S, false>(w, sum, a.nseg, V, u, total);
    } else {
      j = chain_draw<PT, QT, VEC, S, false>(w, sum, a.nseg, V, u, total);
    }
    if (total == 0.0 && e.x >= 0) j = chain_draw_again<PT, QT, VEC, S>(w.p, a.nseg, V, u);
  }
  if (lane == 0) {
    const int n = max(e.a, 0);
    c.emit_len[r] = n + (j >= 0 ? 1 : 0);
    c.status[r] = j >= 0 ? GSE_WALK_OK : GSE_WALK_ERROR;
    c.emit_tokens[r * c.emit_ld + n] = j;
    if (c.emit_probs) c.emit_probs[r * c.emit_ld + n] = j >= 0 ? (float)value<PT>(w.p, j) : 0.0f;
    a.tick[k * a.tstride] = 0;
  }
}

}  // namespace

bool chains_fit(const RowsWs &w, const gsp_chains &c) {  // (the longest segments over the narrowest vectors)
  return (int64_t)c.vocab / (2 * 8 * WAVE) + 1 <= (int64_t)w.rows * w.slices * 64;
}

hipError_t launch_chains(const RowsWs &w, const gsp_chains &c, hipStream_t s) {
  auto go = [&](auto pt, auto qt) {
    constexpr int P = decltype(pt)::value, Q = decltype(qt)::value;
    constexpr int PS = SIZE<P>, QS = Q < 0 ? 0 : SIZE<Q < 0 ? 0 : Q>;
    constexpr int VEC = 16 / (QS > PS ? QS : PS);
    ChainArgs a;
    a.c = c;
    a.sum = w.seg;
    a.tick = w.tick;
    const int64_t nv = (int64_t)c.vocab / VEC;
    const int64_t cap = (int64_t)w.rows * w.slices * 64;         // segment sums that the workspace holds
    const int64_t rows = std::min((int64_t)c.requests, std::min((int64_t)w.ticks, (int64_t)65535));  // requests of a launch, at most
    // One resident round of workgroups over the launch, as long as a wave has a segment; the longest segments that leave every
    // wave one (the last workgroup reads their sums). Where a wave would have eight of the longest or more, four times as
    // many workgroups: rows with and without q even out (512 chains over 262144 bf16 tokens 84 -> 78 us; 64 over 128256 fp32
    // tokens, a segment or two a wave, are slower so: 15.3 -> 21).
    auto segs = [&](int64_t S) { return std::max((int64_t)1, (nv + S * WAVE - 1) / (S * WAVE)); };
    int64_t most = std::max((int64_t)1, std::min((int64_t)(w.round) / rows, (int64_t)WGS_MAX));
    if (segs(8) >= 8 * CW * most) most *= 4;
    int S = 8;
    while (S > 1 && segs(S) < most * CW) S /= 2;
    while (S < 8 && segs(S) > cap) S *= 2;
    a.nseg = (int)segs(S);
    const int64_t wgs = std::min(most, (a.nseg + CW - 1) / (int64_t)CW);
    const int64_t per = std::min(rows, cap / a.nseg);
    // Rows that together pass the last-level cache are read around it. Bytes of one row of p and q a request, us a call over
    // inputs in turn / the same input, cached and around: 134 MB (bf16 128 x 262144) 24.4 / 24.2 and 24.4 / 23.6; 233 MB (fp32
    // 192 x 151936) 41.2 / 31.1 and 37.7 / 35.3; 268 MB (bf16 256 x 262144) 44.7 / 37.0 and 40.5 / 37.5; 311 MB (fp32 256) 53.4 /
    // 44.3 and 48.6 / 46.6; 537 MB (bf16 512) 78.3 / 68.7 and 71.4 / 68.4. Smaller calls lose: 64 fp32 rows 15.0 -> 15.5. So do
    // fp64 rows: 525 MB (256 x 128256) 83.2 / 80.2 and 90.4 / 86.9.
    const bool past = (int64_t)c.requests * c.vocab * (PS + QS) >= (int64_t)256 << 20;
    a.tstride = (int)std::min((int64_t)w.ticks / per, (int64_t)64);
    for (int64_t r0 = 0; r0 < (int64_t)c.requests; r0 += per) {
      a.r0 = (int)r0;
      const dim3 grid((uint32_t)wgs, (uint32_t)std::min(per, (int64_t)c.requests - r0));
      if (S == 1) hipLaunchKernelGGL((chain_kernel<P, Q, 1, false>), grid, dim3(CT), 0, s, a);
      else if (S == 2) hipLaunchKernelGGL((chain_kernel<P, Q, 2, false>), grid, dim3(CT), 0, s, a);
      else if (S == 4) hipLaunchKernelGGL((chain_kernel<P, Q, 4, false>), grid, dim3(CT), 0, s, a);
      else if (!past) hipLaunchKernelGGL((chain_kernel<P, Q, 8, false>), grid, dim3(CT), 0, s, a);
      else hipLaunchKernelGGL((chain_kernel<P, Q, 8, true>), grid, dim3(CT), 0, s, a);
    }
  };
  auto by_q = [&](auto pt) {
    if (!c.draft) return go(pt, std::integral_constant<int, -1>{});
    switch (c.draft_type) {
      case GSP_F64: return go(pt, std::integral_constant<int, GSP_F64>{});
      case GSP_F32: return go(pt, std::integral_constant<int, GSP_F32>{});
      case GSP_BF16: return go(pt, std::integral_constant<int, GSP_BF16>{});
      default: return go(pt, std::integral_constant<int, GSP_F16>{});
    }
  };
  switch (c.target_type) {
    case GSP_F64: by_q(std::integral_constant<int, GSP_F64>{}); break;
    case GSP_F32: by_q(std::integral_constant<int, GSP_F32>{}); break;
    case GSP_BF16: by_q(std::integral_constant<int, GSP_BF16>{}); break;
    default: by_q(std::integral_constant<int, GSP_F16>{}); break;
  }
  return hipGetLastError();
}

}  // namespace gse
