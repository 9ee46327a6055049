// Drafted chains against the target's probability rows (gsp_verify_chains): the accepted length of every request and the
// token drawn after it.
//
// With p_i the target's row after i drafts and q_i the row that draft x_i was drawn from, draft i is accepted iff
// q_i(x_i) > 0 and coin_i q_i(x_i) < p_i(x_i): with probability min(1, p / q). At the first draft a that is not, the token
// comes from max(p_a - q_a, 0), which makes its law p_a again; after the last one from p_n. The tests read two values per
// draft, so what has to be read is one row of p per request, and one of q where a draft was rejected.
#include "gse_dev.h"
#include "gsp_int.h"

namespace gse {

namespace {

constexpr int CT = 256;          // threads of a slice's workgroup
constexpr int CW = CT / WAVE;
constexpr int CS = 8;            // steps that the last slice's search takes at once (CT partial sums each, in LDS)

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
template <int T, int N>
struct Raw {
  static constexpr int W = SIZE<T> * N / 4;
  uint32_t w[W];
  __device__ __forceinline__ void load(const char *row, int64_t t) {
    __builtin_memcpy(w, row + t * SIZE<T>, sizeof w);
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

// The distribution that a request's token is drawn from: weight(t) = max(p(t) - q(t), 0) (Q: q given; X: the draft x's own
// weight dropped, else).
struct ChainRow {
  const char *p, *q;
  int x;
};

// A vector's weights. bad becomes NaN when a weight is not finite (NaN or infinite p or q).
template <int PT, int QT, int VEC>
struct Weights {
  Raw<PT, VEC> p;
  Raw<QT < 0 ? GSP_BF16 : QT, QT < 0 ? 2 : VEC> q;
  __device__ __forceinline__ void load(const ChainRow &w, int64_t t) {
    p.load(w.p, t);
    if constexpr (QT >= 0)
      if (w.q) q.load(w.q, t);
  }
  __device__ __forceinline__ double get(const ChainRow &w, int64_t t, int i, double &bad) const {
    double v = p.get(i);
    if constexpr (QT >= 0) {
      if (w.q) v -= q.get(i);
    } else {
      if (t + i == w.x) v = 0.0;
    }
    bad = fma(v, 0.0, bad);
    return fmax(v, 0.0);
  }
};

// The same for one token.
template <int PT, int QT>
__device__ __forceinline__ double weight(const ChainRow &w, int64_t t, double &bad) {
  double v = value<PT>(w.p, t);
  if constexpr (QT >= 0) {
    if (w.q) v -= value<QT>(w.q, t);
  } else {
    if (t == w.x) v = 0.0;
  }
  bad = fma(v, 0.0, bad);
  return fmax(v, 0.0);
}

struct ChainArgs {
  gsp_chains c;
  int r0;          // first request of the launch
  int ns, steps;   // slices of a row, steps of a slice; a step is one vector a thread
  double *sum;     // [requests of the launch][ns]
  uint32_t *tick;  // [requests of the launch], zero between calls
};

struct ChainShared {
  double part[CS * CT];
  double wave[CW];
  int hit[CW];
  uint32_t ticket;
};

// Sum over the workgroup in a fixed order (every thread gets it).
__device__ __forceinline__ double block_sum(double v, ChainShared &sh) {
  v = wave_sum_f64(v);
  __syncthreads();
  if (lane_id() == 0) sh.wave[threadIdx.x >> 6] = v;
  __syncthreads();
  double t = sh.wave[0];
  for (int k = 1; k < CW; ++k) t += sh.wave[k];
  return t;
}

// This thread's part of the weights of steps [s0, s1) of a row: whole vectors, S at a time, and after the row's last whole
// vector the tokens that are left, one a thread.
// (s1 - s0 is a multiple of S)
template <int PT, int QT, int VEC, int S>
__device__ __forceinline__ double steps_sum(const ChainRow &w, int64_t s0, int64_t s1, int V) {
  const int nv = V / VEC, tid = threadIdx.x;
  double acc = 0.0, bad = 0.0;
  for (int64_t s = s0; s < s1; s += S) {
    Weights<PT, QT, VEC> x[S];
#pragma unroll
    for (int k = 0; k < S; ++k) {
      const int64_t i = (s + k) * CT + tid;  // (past the end: the last vector again, its weights dropped)
      x[k].load(w, min(i, (int64_t)nv - 1) * VEC);
    }
#pragma unroll
    for (int k = 0; k < S; ++k) {
      const int64_t i = (s + k) * CT + tid;
      double a = 0.0;
#pragma unroll
      for (int e = 0; e < VEC; ++e) a += x[k].get(w, min(i, (int64_t)nv - 1) * VEC, e, bad);
      acc += i < nv ? a : 0.0;
    }
  }
  return acc + bad;
}

// The tokens after a row's last whole vector belong to the step after it, as this thread's single token.
template <int PT, int QT, int VEC>
__device__ __forceinline__ double tail_weight(const ChainRow &w, int V) {
  const int t = V / VEC * VEC + (int)threadIdx.x;
  double bad = 0.0;
  const double v = t < V ? weight<PT, QT>(w, t, bad) : 0.0;
  return v + bad;
}

// The first token of steps [s0, s1) (tail: and of the row's tail) with a positive weight whose prefix, from `before` on, reaches
// thr; the last one with a positive weight when rounding leaves none, -1 when there is none at all. By the workgroup.
template <int PT, int QT, int VEC>
__device__ __noinline__ int search(const ChainRow &w, int64_t s0, int64_t s1, bool tail, int V, double before, double thr,
                                   ChainShared &sh) {
  const int nv = V / VEC, tid = threadIdx.x, lane = lane_id(), wv = tid >> 6;
  int last = -1;
  double bad = 0.0;
  for (int64_t s = s0; s < s1; s += CS) {
    // the vectors' sums, then every thread a run of CS of them in vocabulary order
    __syncthreads();
    for (int k = 0; k < CS; ++k) {
      const int64_t i = (s + k) * CT + tid;
      double a = 0.0;
      if (i < nv && s + k < s1) {
        Weights<PT, QT, VEC> x;
        x.load(w, i * VEC);
#pragma unroll
        for (int e = 0; e < VEC; ++e) a += x.get(w, i * VEC, e, bad);
      }
      sh.part[k * CT + tid] = a;
    }
    __syncthreads();
    double run[CS], tot = 0.0;
    for (int k = 0; k < CS; ++k) tot += run[k] = sh.part[tid * CS + k];
    const double inc = wave_incl_scan_f64(tot);
    if (lane == WAVE - 1) sh.wave[wv] = inc;
    __syncthreads();
    double base = before;
    for (int k = 0; k < wv; ++k) base += sh.wave[k];
    const double up = shfl_up_f64(inc, 1);  // (by every lane: a lane that does not take part gives nothing)
    double at = lane > 0 ? base + up : base;
    int hit = -1, pos = -1;  // this thread's first vector that reaches thr, its last with a weight
    double hat = 0.0;
    for (int k = 0; k < CS; ++k) {
      const double nx = at + run[k];
      if (run[k] > 0.0) {
        pos = tid * CS + k;
        if (hit < 0 && !(nx < thr)) {
          hit = pos;
          hat = at;
        }
      }
      at = nx;
    }
    const uint64_t hm = ballot64(hit >= 0), pm = ballot64(pos >= 0);
    // (a thread's run may pass thr where the wave's scan, in another order, had not: the first thread counts)
    const int src = hm ? (int)__builtin_ctzll(hm) : pm ? 63 - (int)__builtin_clzll(pm) : 0;
    const int vec = __shfl(hm ? hit : pos, src, WAVE);
    const double vat = shfl_f64(hat, src);
    for (int k = 0; k < CW; ++k) before += sh.wave[k];
    __syncthreads();
    if (lane == 0) {
      sh.hit[wv] = hm ? vec : pm ? -2 - vec : -1;
      sh.wave[wv] = vat;
    }
    __syncthreads();
    int at_vec = -1;
    double from = 0.0;
    for (int k = CW - 1; k >= 0; --k) {
      if (sh.hit[k] >= 0) {
        at_vec = sh.hit[k];
        from = sh.wave[k];
      }
    }
    int lv = -1;
    for (int k = 0; k < CW; ++k)
      if (sh.hit[k] < -1) lv = -2 - sh.hit[k];
    const int v = at_vec >= 0 ? at_vec : lv;
    if (v >= 0) {  // the vector's tokens, the same in every thread
      const int64_t t0 = (s * CT + v) * VEC;
      Weights<PT, QT, VEC> x;
      x.load(w, t0);
      int found = -1;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const double a = x.get(w, t0, e, bad);
        from += a;
        if (a > 0.0) {
          last = (int)t0 + e;
          if (at_vec >= 0 && found < 0 && !(from < thr)) found = last;
        }
      }
      if (at_vec >= 0) return found >= 0 ? found : last;
    }
  }
  if (tail) {
    for (int t = nv * VEC; t < V; ++t) {
      const double a = weight<PT, QT>(w, t, bad);
      before += a;
      if (a > 0.0) {
        last = t;
        if (!(before < thr)) return t;
      }
    }
  }
  return last;
}

// One workgroup a slice of a request's row: the chain's end (every workgroup finds it: its drafts' values are cached after
// the first), the slice's sum, and the ticket whose last holder searches the row.
template <int PT, int QT, int S>
__global__ __launch_bounds__(CT) void chain_kernel(ChainArgs a) {
  constexpr int VEC = 16 / (QT >= 0 && SIZE<QT < 0 ? 0 : QT> > SIZE<PT> ? SIZE<QT < 0 ? 0 : QT> : SIZE<PT>);
  __shared__ ChainShared sh;
  const gsp_chains &c = a.c;
  const int s = blockIdx.x, k = blockIdx.y, r = a.r0 + k, tid = threadIdx.x, lane = lane_id(), V = (int)c.vocab;
  const ChainEnd e = chain_end<PT, QT>(c, r, s == 0 && tid < WAVE);
  ChainRow w;
  w.p = row_of<PT>(c.target, c.target_ld, e.row);
  w.q = nullptr;
  w.x = -1;
  if (e.x >= 0) {
    if constexpr (QT >= 0) w.q = row_of<QT>(c.draft, c.draft_ld, e.row - r);
    else w.x = e.x;
  }
  const int nv = V / VEC;
  double total = 0.0;
  if (e.a >= 0) {
    const int64_t s0 = (int64_t)s * a.steps;
    double part = nv > 0 ? steps_sum<PT, QT, VEC, S>(w, s0, s0 + a.steps, V) : 0.0;
    if (s == a.ns - 1) part += tail_weight<PT, QT, VEC>(w, V);
    total = block_sum(part, sh);
  }
  double *sum = a.sum + (int64_t)k * a.ns;
  if (tid == 0) {
    st_ag(&sum[s], total);
    store_wait();
    sh.ticket = ticket_add(&a.tick[k]);
  }
  __syncthreads();
  if (sh.ticket != (uint32_t)(a.ns - 1)) return;
  int j = -1;
  if (e.a >= 0) {
    total = 0.0;
    for (int i0 = 0; i0 < a.ns; i0 += WAVE) total += wave_sum_f64(i0 + lane < a.ns ? ld_ag(&sum[i0 + lane]) : 0.0);
    int64_t s0 = 0, s1 = (int64_t)a.ns * a.steps;
    bool tail = true;
    double before = 0.0, thr = 0.0;
    if (total == 0.0 && e.x >= 0) {  // p is nowhere above q: drawn from p itself, by this workgroup alone
      w.q = nullptr;
      w.x = -1;
      total = block_sum((nv > 0 ? steps_sum<PT, QT, VEC, S>(w, s0, s1, V) : 0.0) + tail_weight<PT, QT, VEC>(w, V), sh);
      thr = c.u[r] * total;
    } else if (total > 0.0) {
      thr = c.u[r] * total;
      int at = -1, lst = -1;  // the slice that the draw falls into
      double lb = 0.0;
      for (int i0 = 0; i0 < a.ns && at < 0; i0 += WAVE) {
        const double x = i0 + lane < a.ns ? ld_ag(&sum[i0 + lane]) : 0.0;
        const double inc = before + wave_incl_scan_f64(x);
        const uint64_t hit = ballot64(x > 0.0 && !(inc < thr)), pos = ballot64(x > 0.0);
        if (hit) {
          const int l = (int)__builtin_ctzll(hit);
          at = i0 + l;
          if (l > 0) before = shfl_f64(inc, l - 1);
        } else {
          if (pos) {
            const int l = 63 - (int)__builtin_clzll(pos);
            lst = i0 + l;
            lb = l > 0 ? shfl_f64(inc, l - 1) : before;
          }
          before = shfl_f64(inc, WAVE - 1);
        }
      }
      if (at < 0) {
        at = lst;
        before = lb;
      }
      s0 = (int64_t)at * a.steps;
      s1 = s0 + a.steps;
      tail = at == a.ns - 1;
    }
    if (total > 0.0 && total < INFINITY) j = search<PT, QT, VEC>(w, s0, s1, tail, V, before, thr, sh);
  }
  if (tid == 0) {
    const int n = max(e.a, 0);
    c.emit_len[r] = n + (j >= 0 ? 1 : 0);
    c.status[r] = j >= 0 ? GSE_WALK_OK : GSE_WALK_ERROR;
    c.emit_tokens[r * c.emit_ld + n] = j;
    if (c.emit_probs) c.emit_probs[r * c.emit_ld + n] = j >= 0 ? (float)value<PT>(w.p, j) : 0.0f;
    a.tick[k] = 0;
  }
}

}  // namespace

hipError_t launch_chains(const RowsWs &w, const gsp_chains &c, hipStream_t s) {
  auto go = [&](auto pt, auto qt) {
    constexpr int P = decltype(pt)::value, Q = decltype(qt)::value;
    constexpr int PS = SIZE<P>, QS = Q < 0 ? 0 : SIZE<Q < 0 ? 0 : Q>;
    constexpr int VEC = 16 / (QS > PS ? QS : PS);
    ChainArgs a;
    a.c = c;
    a.sum = w.seg;
    a.tick = w.tick;
    const int64_t all = ((int64_t)c.vocab / VEC + CT - 1) / CT;  // steps of a row (0: the tail alone)
    const int64_t cap = (int64_t)w.rows * w.slices * 64;         // slice sums that the workspace holds
    const int64_t most = min((int64_t)w.rows, (int64_t)65535);   // requests of a launch
    const int64_t rows = min((int64_t)c.requests, most);
    // The steps of a slice: as few as keep the launch at two resident rounds of workgroups.
    int64_t steps = 1;
    while (steps < 8 && rows * ((all + steps - 1) / steps) > 2 * (int64_t)w.round) steps *= 2;
    while ((all + steps - 1) / steps > cap) steps *= 2;
    a.steps = (int)steps;
    a.ns = (int)max((int64_t)1, (all + steps - 1) / steps);
    const int64_t per = min(rows, cap / a.ns);
    for (int64_t r0 = 0; r0 < (int64_t)c.requests; r0 += per) {
      a.r0 = (int)r0;
      const dim3 grid((uint32_t)a.ns, (uint32_t)min(per, (int64_t)c.requests - r0));
      if (steps == 1) hipLaunchKernelGGL((chain_kernel<P, Q, 1>), grid, dim3(CT), 0, s, a);
      else if (steps == 2) hipLaunchKernelGGL((chain_kernel<P, Q, 2>), grid, dim3(CT), 0, s, a);
      else if (steps == 4) hipLaunchKernelGGL((chain_kernel<P, Q, 4>), grid, dim3(CT), 0, s, a);
      else hipLaunchKernelGGL((chain_kernel<P, Q, 8>), grid, dim3(CT), 0, s, a);
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
