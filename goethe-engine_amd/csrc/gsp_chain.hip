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

constexpr int CT = 256;          // threads of a request's workgroup
constexpr int CW = CT / WAVE;

// One value of a row of type T as fp64 (exact for every type).
template <int T>
__device__ __forceinline__ double value(const void *row, int64_t t) {
  if constexpr (T == GSP_F64) return ((const double *)row)[t];
  else if constexpr (T == GSP_F32) return (double)((const float *)row)[t];
  else if constexpr (T == GSP_BF16) return (double)bf16_to_f32(((const uint16_t *)row)[t]);
  else return (double)((const _Float16 *)row)[t];
}
template <int T>
constexpr int SIZE = T == GSP_F64 ? 8 : T == GSP_F32 ? 4 : 2;
template <int T>
__device__ __forceinline__ const char *row_of(const void *base, int64_t ld, int64_t row) {
  return (const char *)base + row * ld * SIZE<T>;
}

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
  const int b0 = c.begin[r], b1 = c.begin[r + 1];
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
      const int xf = __shfl(x, f, WAVE);
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

struct ChainShared {
  ChainEnd e;
  double sum[CW];
  int hit[CW];
};

// The weight of token t, NaN where it is not finite.
template <int PT, int QT>
__device__ __forceinline__ double weight(const char *p, const char *q, int x, int t) {
  double v = value<PT>(p, t);
  if constexpr (QT >= 0) {
    if (q) v -= value<QT>(q, t);
  } else {
    if (t == x) v = 0.0;
  }
  const double bad = v * 0.0;
  return (v > 0.0 ? v : 0.0) + bad;
}

__device__ __forceinline__ double block_sum(double v, ChainShared &sh) {
  v = wave_sum_f64(v);
  __syncthreads();
  if (lane_id() == 0) sh.sum[threadIdx.x >> 6] = v;
  __syncthreads();
  double t = sh.sum[0];
  for (int k = 1; k < CW; ++k) t += sh.sum[k];
  return t;
}

// One workgroup a request: the row's sum, then its walk in vocabulary order, CT tokens at a time.
template <int PT, int QT>
__global__ __launch_bounds__(CT) void chain_kernel(gsp_chains c) {
  __shared__ ChainShared sh;
  const int r = blockIdx.x, tid = threadIdx.x, lane = lane_id(), w = tid >> 6, V = (int)c.vocab;
  if (w == 0) {
    const ChainEnd e = chain_end<PT, QT>(c, r, true);
    if (lane == 0) sh.e = e;
  }
  __syncthreads();
  const ChainEnd e = sh.e;
  int j = -1;
  const char *p = row_of<PT>(c.target, c.target_ld, e.row);
  if (e.a >= 0) {
    const char *q = QT >= 0 && e.x >= 0 ? row_of<QT < 0 ? GSP_F32 : QT>(c.draft, c.draft_ld, e.row - r) : nullptr;
    int x = e.x;
    double total = 0.0;
    for (int go = 0; go < 2; ++go) {
      double s = 0.0;
      for (int64_t t = tid; t < V; t += CT) s += weight<PT, QT>(p, q, x, (int)t);
      total = block_sum(s, sh);
      if (total != 0.0 || e.x < 0) break;
      q = nullptr;  // (p is nowhere above q: drawn from p itself)
      x = -1;
    }
    if (total > 0.0 && total < INFINITY) {
      const double thr = c.u[r] * total;
      double before = 0.0;
      int last = -1;
      for (int64_t t0 = 0; t0 < V && j < 0; t0 += CT) {
        const int t = (int)(t0 + tid);
        const double v = t < V ? weight<PT, QT>(p, q, x, t) : 0.0;
        const double inc = wave_incl_scan_f64(v);
        __syncthreads();
        if (lane == WAVE - 1) sh.sum[w] = inc;
        __syncthreads();
        double base = before;
        for (int k = 0; k < w; ++k) base += sh.sum[k];
        const uint64_t pos = ballot64(v > 0.0), at = ballot64(v > 0.0 && !(base + inc < thr));
        const int64_t tw = t0 + w * WAVE;
        if (lane == 0) sh.hit[w] = at ? (int)(tw + __builtin_ctzll(at)) : pos ? (int)(-2 - (tw + 63 - __builtin_clzll(pos))) : -1;
        for (int k = 0; k < CW; ++k) before += sh.sum[k];
        __syncthreads();
        for (int k = 0; k < CW && j < 0; ++k) {
          if (sh.hit[k] >= 0) j = sh.hit[k];
          else if (sh.hit[k] < -1) last = -2 - sh.hit[k];
        }
      }
      if (j < 0) j = last;
    }
  }
  if (tid == 0) {
    const int a = max(e.a, 0);
    c.emit_len[r] = a + (j >= 0 ? 1 : 0);
    c.status[r] = j >= 0 ? GSE_WALK_OK : GSE_WALK_ERROR;
    c.emit_tokens[r * c.emit_ld + a] = j;
    if (c.emit_probs) c.emit_probs[r * c.emit_ld + a] = j >= 0 ? (float)value<PT>(p, j) : 0.0f;
  }
}

}  // namespace

hipError_t launch_chains(const RowsWs &w, const gsp_chains &c, hipStream_t s) {
  (void)w;
  auto go = [&](auto pt, auto qt) {
    hipLaunchKernelGGL((chain_kernel<decltype(pt)::value, decltype(qt)::value>), dim3(c.requests), dim3(CT), 0, s, c);
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
