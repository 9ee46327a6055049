// Beam search's selection (gsk_beam, include/gsk.h): for each request the n best of score + log softmax over its beams and the
// vocabulary.
//
// One pass over the logits. A row is cut into slices of BS tokens, one a workgroup, held in registers. The slice's n largest: in
// each of the four waves, a quarter of n lanes' maxima (rounded up) reach some value, so n elements reach the least of the four;
// the elements that reach it are listed (a few more than n in an unordered row) and ranked by counting; where more tie with the
// bound than the list holds, the n-th largest (value, token) is found digit by digit instead. The slice leaves its maximum m, its
// sum of exp(x - m) and its list. The sum decides the order of tokens of different beams, so the large terms, the listed ones,
// are fp64; the many small ones are fp32 in each thread (their errors average out: about 1e-9 of the sum) and fp64 from there on.
// The last workgroup of a request (a ticket) joins its beams' slices: log of each beam's sum, then the n best of all lists by the
// same two steps over the lists' heads.
#include "gsk_dev.h"
#include "gsk_int.h"

#include <float.h>

namespace gse {

namespace {

constexpr int BT = 256;
constexpr uint32_t BS = 8192;      // tokens of a slice
constexpr int BE = BS / BT;        // a thread's elements
constexpr uint32_t BL = 1024;      // entries of the list
constexpr uint32_t BLISTS = GSK_MAX_BEAMS;

struct SliceSum {  // a slice's part of its row's sum
  double sum;
  float max;
  uint32_t bad;  // a +inf among the logits
};

struct BeamShared {
  uint64_t list[BL];
  uint64_t sub[BL];  // (the join: the entries' places)
  double red[BT / WAVE];
  uint64_t redu[BT / WAVE];
  uint32_t hist[256];
  uint32_t n, last, rank;
  double base[BLISTS], shift[BLISTS];  // a beam's maximum; log of its sum
  double score[BLISTS];
};

__device__ __forceinline__ float load_logit(const void *p, uint32_t type, int64_t i) {
  if (type == GSK_F32) return ((const float *)p)[i];
  if (type == GSK_BF16) return bf16_to_f32(((const uint16_t *)p)[i]);
  return (float)((const _Float16 *)p)[i];
}

__device__ __forceinline__ double block_sum_f64(double v, double *red) {
  v = wave_sum_f64(v);
  __syncthreads();
  if (lane_id() == 0) red[threadIdx.x / WAVE] = v;
  __syncthreads();
  double s = 0;
  for (int i = 0; i < BT / WAVE; ++i) s += red[i];
  return s;
}
__device__ __forceinline__ uint64_t block_max_u64(uint64_t v, uint64_t *red) {
  v = wave_max_u64(v);
  __syncthreads();
  if (lane_id() == 0) red[threadIdx.x / WAVE] = v;
  __syncthreads();
  uint64_t s = 0;
  for (int i = 0; i < BT / WAVE; ++i) s = max(s, red[i]);
  return s;
}

// The k-th largest of the workgroup's values, one a thread (1 <= k <= BT); through LDS.
__device__ __forceinline__ uint32_t block_kth_u32(uint32_t v, uint32_t k, uint32_t *all) {
  __syncthreads();
  all[threadIdx.x] = v;
  __syncthreads();
  uint32_t o[BT / WAVE], r = 0;
  for (int i = 0; i < BT / WAVE; ++i) o[i] = all[i * WAVE + lane_id()];
  for (int b = 31; b >= 0; --b) {
    const uint32_t c = r | (1u << b);
    uint32_t n = 0;
    for (int i = 0; i < BT / WAVE; ++i) n += (uint32_t)__popcll(ballot64(o[i] >= c));
    if (n >= k) r = c;
  }
  return r;
}

// A total order of doubles as unsigned integers (no NaNs).
__device__ __forceinline__ uint64_t dkey(double d) {
  const uint64_t b = (uint64_t)__double_as_longlong(d + 0.0);  // (-0 -> 0)
  return b >> 63 ? ~b : b | 0x8000000000000000ull;
}
__device__ __forceinline__ double dkey_inv(uint64_t k) {
  return __longlong_as_double((long long)(k >> 63 ? k & 0x7FFFFFFFFFFFFFFFull : ~k));
}

template <uint32_t T, bool WIDE>
__global__ __launch_bounds__(BT) void beam_kernel(gsk_beams a, uint32_t slices, uint32_t *tick, uint32_t r0) {
  __shared__ BeamShared sh;
  const uint32_t tid = threadIdx.x, slice = blockIdx.x, beam = blockIdx.y % a.beams, r = r0 + blockIdx.y / a.beams;
  const uint32_t row = r * a.beams + beam, n = a.n;
  const int64_t lists = (int64_t)a.requests * a.beams * slices;
  SliceSum *sums = (SliceSum *)a.work;
  uint64_t *tops = (uint64_t *)(sums + lists);
  // the slice's elements, -inf for NaN and past the row
  float v[BE];
  const char *x = (const char *)a.logits + (int64_t)row * a.ld * type_size<T>;
  const uint32_t t0 = slice * BS;
  constexpr int VE = WIDE ? 8 : 1;  // elements of a load
  auto token = [&](int e) { return t0 + (uint32_t)(e / VE) * (BT * VE) + tid * VE + (uint32_t)(e % VE); };
  if (WIDE && t0 + BS <= a.vocab) {
#pragma unroll
    for (int e = 0; e < BE; e += 8) to_f32(load_raw8<T>(x + (int64_t)token(e) * type_size<T>), *(float(*)[8])(v + e));
  } else {
#pragma unroll
    for (int e = 0; e < BE; ++e) v[e] = token(e) < a.vocab ? load_logit(x, T, token(e)) : -INFINITY;
  }
  float top = -INFINITY;
#pragma unroll
  for (int e = 0; e < BE; ++e) {
    v[e] = fmaxf(v[e], -INFINITY);
    top = fmaxf(top, v[e]);
  }
  // each wave's bound, of the values' upper 16 bits; the slice's maximum
  const uint32_t own = fkey(top) >> 16, kth = wave_kth_largest_u16(own, (int)(n + 3) / 4) << 16, most = wave_max_u32(fkey(top));
  if (lane_id() == 0) sh.redu[tid / WAVE] = (uint64_t)most << 32 | kth;
  if (tid == 0) sh.n = 0;
  __syncthreads();
  uint32_t best = 0, bound_key = ~0u;
#pragma unroll
  for (int i = 0; i < BT / WAVE; ++i) {
    best = max(best, (uint32_t)(sh.redu[i] >> 32));
    bound_key = min(bound_key, (uint32_t)sh.redu[i]);
  }
  const float m = fkey_inv(best);
  const bool some = best > KEY_NEGINF && best < KEY_POSINF;  // (+inf: the row gives nothing)
  const float bound = bound_key > KEY_NEGINF ? fkey_inv(bound_key) : -FLT_MAX;
  auto term = [&](float y) { return __builtin_amdgcn_exp2f((y - m) * 1.44269504f); };
  double sum = 0;
  if (some) {
    float rest = 0;
#pragma unroll
    for (int e = 0; e < BE; ++e) {
      rest += term(v[e]);
      if (v[e] >= bound) {
        const uint32_t k = atomicAdd(&sh.n, 1u);
        if (k < BL) sh.list[k] = pack(fkey(v[e]), token(e));
      }
    }
    sum = rest;
  }
  __syncthreads();
  uint32_t count = sh.n;
  if (count > BL) {
    // the n-th largest (value, token), 8 bits at a time
    uint64_t prefix = 0;
    uint32_t want = n;
    for (int shift = 56; shift >= 0; shift -= 8) {
      __syncthreads();
      sh.hist[tid] = 0;
      __syncthreads();
#pragma unroll
      for (int e = 0; e < BE; ++e) {
        const uint64_t p = pack(fkey(v[e]), token(e));
        if (v[e] >= bound && (shift == 56 || (p >> (shift + 8)) == (prefix >> (shift + 8))))
          atomicAdd(&sh.hist[(p >> shift) & 255], 1u);
      }
      __syncthreads();
      if (tid == 0) {
        uint32_t above = 0;
        int d = 255;
        while (d > 0 && above + sh.hist[d] < want) above += sh.hist[d--];
        sh.rank = want - above;
        sh.last = (uint32_t)d;
      }
      __syncthreads();
      want = sh.rank;
      prefix |= (uint64_t)sh.last << shift;
    }
    if (tid == 0) sh.n = 0;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < BE; ++e) {
      const uint64_t p = pack(fkey(v[e]), token(e));
      if (v[e] >= bound && p >= prefix) sh.list[atomicAdd(&sh.n, 1u)] = p;
    }
    __syncthreads();
    count = sh.n;
  }
  uint64_t *out = tops + ((int64_t)row * slices + slice) * n;
  for (uint32_t i = tid; i < count; i += BT) {
    const uint64_t p = sh.list[i];
    sum += exp((double)fkey_inv(pk_key(p)) - (double)m) - (double)term(fkey_inv(pk_key(p)));
    uint32_t rank = 0;
    for (uint32_t k = 0; k < count; ++k) rank += sh.list[k] > p;
    if (rank < n) st_ag(out + rank, p);
  }
  for (uint32_t i = count + tid; i < n; i += BT) st_ag(out + i, (uint64_t)0);
  sum = block_sum_f64(sum, sh.red);
  if (tid == 0) {
    SliceSum *o = sums + (int64_t)row * slices + slice;
    st_ag((uint64_t *)&o->sum, (uint64_t)__double_as_longlong(some ? sum : 0.0));
    st_ag((uint64_t *)&o->max, (uint64_t)__float_as_uint(some ? m : -INFINITY) | (uint64_t)(best >= KEY_POSINF) << 32);
  }
  store_wait();
  __syncthreads();
  if (tid == 0) sh.last = ticket_add(tick + blockIdx.y / a.beams) == a.beams * slices - 1;
  __syncthreads();
  if (!sh.last) return;
  if (tid == 0) st_ag(tick + blockIdx.y / a.beams, 0u);

  // ---- the join: a thread a list (a slice of a beam), in turn -------------------------------------------------------------
  const uint32_t total = a.beams * slices, lane = lane_id(), wave = tid / WAVE;
  const SliceSum *my = sums + (int64_t)r * total;
  const uint64_t *heads = tops + (int64_t)r * total * n;
  for (uint32_t b = wave; b < a.beams; b += BT / WAVE) {
    float bm = -INFINITY;
    uint32_t bad = 0;
    for (uint32_t i = lane; i < slices; i += WAVE) {
      const uint64_t v = ld_ag((const uint64_t *)&my[b * slices + i].max);
      bm = fmaxf(bm, __uint_as_float((uint32_t)v));
      bad |= (uint32_t)(v >> 32);
    }
    bm = wave_max_f32(bm);
    bad = ballot64(bad != 0) != 0;
    double s = 0;
    for (uint32_t i = lane; i < slices; i += WAVE) {
      const double part = __longlong_as_double((long long)ld_ag((const uint64_t *)&my[b * slices + i].sum));
      const float pm = __uint_as_float((uint32_t)ld_ag((const uint64_t *)&my[b * slices + i].max));
      if (part > 0) s += part * exp((double)pm - (double)bm);
    }
    s = wave_sum_f64(s);
    const float score = a.scores[(int64_t)r * a.beams + b];
    if (lane == 0) {
      const bool ok = !bad && bm > -INFINITY && isfinite(score);
      sh.base[b] = ok ? (double)bm : -INFINITY;  // (-inf: the beam gives nothing)
      sh.shift[b] = ok ? log(s) : 0.0;
      sh.score[b] = ok ? (double)score : 0.0;
    }
  }
  __syncthreads();
  auto value = [&](uint32_t list, uint64_t p) -> uint64_t {  // 0: none
    const uint32_t b = list / slices;
    if (p == 0 || sh.base[b] == -INFINITY) return 0;
    return dkey(((double)fkey_inv(pk_key(p)) - sh.base[b]) - sh.shift[b] + sh.score[b]);
  };
  // a bound that n entries reach: the n-th largest of the threads' largest heads, by its upper 32 bits
  uint64_t lead = 0;
  for (uint32_t i = tid; i < total; i += BT) lead = max(lead, value(i, ld_ag(heads + (int64_t)i * n)));
  const uint64_t from = max((uint64_t)block_kth_u32((uint32_t)(lead >> 32), n, (uint32_t *)sh.list) << 32, (uint64_t)1);
  if (tid == 0) sh.n = 0;
  __syncthreads();
  for (uint32_t i = tid; i < total; i += BT) {
    for (uint32_t k = 0; k < n; ++k) {
      const uint64_t p = ld_ag(heads + (int64_t)i * n + k), v = value(i, p);
      if (v < from) break;  // (a list descends)
      const uint32_t at = atomicAdd(&sh.n, 1u);
      if (at < BL) {
        sh.list[at] = v;
        sh.sub[at] = (uint64_t)(i / slices) << 32 | pk_id(p);
      }
    }
  }
  __syncthreads();
  count = sh.n;
  int32_t *tokens = a.tokens + (int64_t)r * n, *parents = a.parents + (int64_t)r * n;
  float *scores = a.out_scores + (int64_t)r * n;
  auto emit = [&](uint32_t rank, uint64_t v, uint64_t place) {
    tokens[rank] = v ? (int32_t)(uint32_t)place : -1;
    parents[rank] = v ? (int32_t)(place >> 32) : -1;
    scores[rank] = v ? (float)dkey_inv(v) : -INFINITY;
  };
  if (count <= BL) {
    for (uint32_t i = tid; i < count; i += BT) {
      const uint64_t v = sh.list[i], p = sh.sub[i];
      uint32_t rank = 0;
      for (uint32_t k = 0; k < count; ++k) rank += sh.list[k] > v || (sh.list[k] == v && sh.sub[k] < p);
      if (rank < n) emit(rank, v, p);
    }
    for (uint32_t i = count + tid; i < n; i += BT) emit(i, 0, 0);
    return;
  }
  // more entries than the list holds: one after the other, the largest that comes after the last one taken
  uint64_t lv = ~0ull, lp = 0;
  for (uint32_t k = 0; k < n; ++k) {
    uint64_t bv = 0, bp = ~0ull;
    for (uint32_t i = tid; i < total; i += BT) {
      for (uint32_t e = 0; e < n; ++e) {
        const uint64_t p = ld_ag(heads + (int64_t)i * n + e), v = value(i, p);
        if (v == 0 || v < bv) break;
        const uint64_t place = (uint64_t)(i / slices) << 32 | pk_id(p);
        if ((v < lv || (v == lv && k > 0 && place > lp)) && (v > bv || place < bp)) {
          bv = v;
          bp = place;
        }
      }
    }
    const uint64_t v = block_max_u64(bv, sh.redu), p = ~block_max_u64(bv == v && v ? ~bp : 0, sh.redu);
    if (tid == 0) emit(k, v, p);
    lv = v;
    lp = p;
    if (v == 0) {
      for (uint32_t i = k + 1 + tid; i < n; i += BT) emit(i, 0, 0);
      return;
    }
  }
}

}  // namespace

uint32_t beam_slices(const gsk_beams &a) { return (a.vocab + BS - 1) / BS; }

int64_t beam_work(const gsk_beams &a) {
  return (int64_t)a.requests * a.beams * beam_slices(a) * (int64_t)(sizeof(SliceSum) + a.n * sizeof(uint64_t));
}

hipError_t launch_beam(const gsk_beams &a, uint32_t *tick, uint32_t tickets, hipStream_t s) {
  const uint32_t slices = beam_slices(a);
  // a launch takes a ticket per request, and 65535 rows at most
  const uint32_t most = min(tickets, 65535u / a.beams);
  auto go = [&](auto type, auto wide) {
    for (uint32_t r0 = 0; r0 < a.requests; r0 += most)
      hipLaunchKernelGGL((beam_kernel<type(), wide()>), dim3(slices, min(most, a.requests - r0) * a.beams), dim3(BT), 0, s, a, slices,
                         tick, r0);
  };
  const uint64_t size = a.type == GSK_F32 ? 4 : 2;
  const bool wide = ((uint64_t)a.logits | (uint64_t)a.ld * size) % 16 == 0;
  auto by = [&](auto type) {
    if (wide) go(type, std::true_type{});
    else go(type, std::false_type{});
  };
  if (a.type == GSK_F32) by(std::integral_constant<uint32_t, GSK_F32>{});
  else if (a.type == GSK_BF16) by(std::integral_constant<uint32_t, GSK_BF16>{});
  else by(std::integral_constant<uint32_t, GSK_F16>{});
  return hipGetLastError();
}

}  // namespace gse
