// Beam search's selection (gsk_beam, include/gsk.h): for each request the n best of score + log softmax over its beams and the
// vocabulary.
//
// One pass over the logits. A row is cut into slices of BS tokens, held in registers; a workgroup takes one or more slices of a
// row in turn (the next one's loads in flight) and keeps the n largest so far. A slice's n largest: in each of the four waves, a
// quarter of n lanes' maxima (rounded up) reach some value, so n elements reach the least of the four; the elements that reach
// it, and the n-th largest of the slices before, are listed (a few more than n in an unordered row) and ranked by counting; where
// more tie with the bound than the list holds, the n-th largest (value, token) is found digit by digit instead. The workgroup
// leaves its maximum m, its sum of exp(x - m) and its list. The sum decides the order of tokens of different beams: a term is exp2 in
// fp32, off by 2^-24 (2 |x - m| + 4) of it at most and by either sign, added up in fp64; the listed ones, the largest, are corrected to
// fp64 (by whole multiples of 2^-62: in any order the same, so that equal rows have equal sums). Measured over rows of 128256 logits,
// fp32, bfloat16 and float16, normal (sigma 1 to 5), uniform and with one peak: 5e-9 of the sum at most (a thread's terms of a slice added
// up in fp32: 5e-8, beside a peak 1e-6; 64 x 8 rows took 64 us instead of 66). The last workgroup of a request (a ticket) joins its beams'
// lists: log of each beam's sum, then the n best of all entries by the same two steps.
//
// Bound: 4 beams of 128256 fp32 logits, 14.4 us, are a chain: a slice's load, its maxima, bound, list and ranks (8 us), the ticket, the
// join's reads, logs and ranks. 64 requests of 8 beams of 151936 bf16 logits (156 MB), 66 us or 2.4 TB/s, are bound by what waves wait
// for, 54 % of their cycles by the counters (three barriers a slice, the list and its ranks; the last request's join), then by
// instructions (17 on each element of 2 bytes: unpacking, maxima, exp2, its sum in fp64, compare).
#include "gsk_dev.h"
#include "gsk_int.h"

#include <float.h>

namespace gse {

namespace {

constexpr int BT = 256;
constexpr uint32_t BS = 8192;      // tokens of a slice
constexpr int BE = BS / BT;        // a thread's elements
constexpr uint32_t BL = 1024;      // entries of the list
constexpr uint32_t LISTS = 1024;   // a request's lists, at most
constexpr float LOG2E = 0x1.715476p+0f, LOG2E_REST = 0x1.4ae0cp-26f;
constexpr int AHEAD = 8;           // entries of its request's lists that a thread reads at once in the join

struct ListSum {  // a workgroup's part of its row's sum
  double sum;
  float max;
  uint32_t bad;  // a +inf among the logits
};

struct BeamShared {
  uint64_t list[BL];
  union {
    uint64_t sub[BL];                 // (the join: the entries' places)
    double sums[LISTS];               // (before that: the lists' sums)
  };
  uint64_t best[GSK_MAX_KEEP];        // the n largest so far
  float maxs[LISTS];                  // the join: the lists' maxima (NaN: a +inf in the row)
  double red[BT / WAVE];
  uint64_t redu[BT / WAVE];
  uint32_t hist[256];
  unsigned long long fix;             // the listed terms' fp64 values less their fp32 ones, in units of 2^-62
  uint32_t n, last, rank;
  double base[GSK_MAX_BEAMS], shift[GSK_MAX_BEAMS], score[GSK_MAX_BEAMS];  // a beam's maximum, log of its sum, score
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
__global__ __launch_bounds__(BT, 4) void beam_kernel(gsk_beams a, uint32_t parts, Div by_beam, uint32_t *tick, uint32_t r0) {
  __shared__ BeamShared sh;
  const uint32_t tid = threadIdx.x, part = blockIdx.x, beam = blockIdx.y % a.beams, r = r0 + blockIdx.y / a.beams;
  const uint32_t row = r * a.beams + beam, n = a.n, lane = lane_id(), wave = tid / WAVE;
  ListSum *sums = (ListSum *)a.work;
  uint64_t *tops = (uint64_t *)(sums + (int64_t)a.requests * a.beams * parts);
  const char *x = (const char *)a.logits + (int64_t)row * a.ld * type_size<T>;
  const uint32_t slices = (a.vocab + BS - 1) / BS, first = (uint32_t)((uint64_t)slices * part / parts);
  const uint32_t end = (uint32_t)((uint64_t)slices * (part + 1) / parts);
  constexpr int VE = WIDE ? 8 : 1;  // elements of a load
  // a slice's elements as they are, 16 bytes a load (unaligned rows: one by one), -inf past the row
  Raw8<T> raw[BE / 8];
  float v[BE];
  auto token = [&](uint32_t slice, int e) { return slice * BS + (uint32_t)(e / VE) * (BT * VE) + tid * VE + (uint32_t)(e % VE); };
  constexpr uint32_t NOTHING = T == GSK_F32 ? 0xFF800000u : T == GSK_BF16 ? 0xFF80FF80u : 0xFC00FC00u;
  auto load = [&](uint32_t slice) {
#pragma unroll
    for (int e = 0; WIDE && e < BE; e += 8) {
#pragma unroll
      for (int i = 0; i < Raw8<T>::N; ++i) raw[e / 8].w[i] = NOTHING;
      if (token(slice, e) + 8 <= a.vocab) raw[e / 8] = load_raw8<T>(x + (int64_t)token(slice, e) * type_size<T>);
    }
  };
  load(first);
  uint32_t kept = 0;          // entries of sh.best
  uint32_t top_key = 0;       // of the slices before: their largest value ...
  float top = -INFINITY;
  double sum = 0;             // ... and the thread's part of the sum of exp(x - it)
  auto settle = [&] {         // the listed terms of the slice before (thread 0; after a barrier)
    sum += (double)(long long)sh.fix * 0x1p-62;
    sh.fix = 0;
  };
  if (tid == 0) sh.fix = 0;
  for (uint32_t slice = first; slice < end; ++slice) {
#pragma unroll
    for (int e = 0; e < BE; e += 8) {
      if constexpr (WIDE) to_f32(raw[e / 8], *(float(*)[8])(v + e));
      const bool some = WIDE ? token(slice, e) < a.vocab && token(slice, e) + 8 > a.vocab : true;  // (the row's ragged end)
      if (some) {
#pragma unroll
        for (int i = e; i < e + 8; ++i) v[i] = token(slice, i) < a.vocab ? load_logit(x, T, token(slice, i)) : -INFINITY;
      }
    }
    if (slice + 1 < end) load(slice + 1);
    float of8[BE / 8], most = -INFINITY;
#pragma unroll
    for (int e = 0; e < BE; ++e) {
      v[e] = fmaxf(v[e], -INFINITY);  // (NaN counts as -inf)
      of8[e / 8] = e % 8 ? fmaxf(of8[e / 8], v[e]) : v[e];
    }
#pragma unroll
    for (int e = 0; e < BE / 8; ++e) most = fmaxf(most, of8[e]);
    // each wave's bound, of the values' upper 16 bits; the slice's maximum
    const uint32_t kth = wave_kth_largest_u16(fkey(most) >> 16, (int)(n + 3) / 4) << 16, wave_most = wave_max_u32(fkey(most));
    __syncthreads();  // (the slice before is done with the list)
    if (lane == 0) sh.redu[wave] = (uint64_t)wave_most << 32 | kth;
    if (tid < kept) sh.list[tid] = sh.best[tid];
    if (tid == 0) {
      sh.n = kept;
      settle();
    }
    __syncthreads();
    uint32_t bound_key = ~0u, now_key = top_key;
#pragma unroll
    for (int i = 0; i < BT / WAVE; ++i) {
      now_key = max(now_key, (uint32_t)(sh.redu[i] >> 32));
      bound_key = min(bound_key, (uint32_t)sh.redu[i]);
    }
    if (kept == n) bound_key = max(bound_key, pk_key(sh.best[n - 1]));
    const float now = fkey_inv(now_key);
    if (now_key > top_key && top_key > KEY_NEGINF) sum *= exp((double)top - (double)now);
    top_key = now_key;
    top = now;
    if (now_key <= KEY_NEGINF || now_key >= KEY_POSINF) continue;  // (nothing yet; or +inf: the row gives nothing)
    const float bound = bound_key > KEY_NEGINF ? fkey_inv(bound_key) : -FLT_MAX;
    auto term = [&](float y) {  // (log2 e as two numbers, so that a term's error has either sign)
      const float d = y - now;
      return __builtin_amdgcn_exp2f(__builtin_fmaf(d, LOG2E, d * LOG2E_REST));
    };
#pragma unroll
    for (int g = 0; g < BE / 8; ++g) {
      if (ballot64(of8[g] >= bound) == 0) continue;  // (after a row's first slice most have none)
#pragma unroll
      for (int e = 8 * g; e < 8 * g + 8; ++e) {
        if (v[e] >= bound) {
          const uint32_t k = atomicAdd(&sh.n, 1u);
          if (k < BL) sh.list[k] = pack(fkey(v[e]), token(slice, e));
        }
      }
    }
    double odd = 0;  // (fp64 from the first term on: small ones next to a large one are not lost)
#pragma unroll
    for (int e = 0; e < BE; e += 2) {
      sum += (double)term(v[e]);
      odd += (double)term(v[e + 1]);
    }
    sum += odd;
    __syncthreads();
    uint32_t count = sh.n;
    if (count > BL) {
      // the slice's n-th largest (value, token), 8 bits at a time; read again, so that the rare path needs no registers
      auto entry = [&](int e) {
        const uint32_t t = slice * BS + e * BT + tid;
        const float y = t < a.vocab ? fmaxf(load_logit(x, T, t), -INFINITY) : -INFINITY;
        return y >= bound ? pack(fkey(y), t) : (uint64_t)0;
      };
      uint64_t prefix = 0;
      uint32_t want = n;
      for (int shift = 56; shift >= 0; shift -= 8) {
        __syncthreads();
        sh.hist[tid] = 0;
        __syncthreads();
#pragma unroll 1
        for (int e = 0; e < BE; ++e) {
          const uint64_t p = entry(e);
          if (p && (shift == 56 || (p >> (shift + 8)) == (prefix >> (shift + 8)))) atomicAdd(&sh.hist[(p >> shift) & 255], 1u);
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
      if (tid == 0) sh.n = kept;
      __syncthreads();
#pragma unroll 1
      for (int e = 0; e < BE; ++e) {
        const uint64_t p = entry(e);
        if (p >= prefix) sh.list[atomicAdd(&sh.n, 1u)] = p;
      }
      __syncthreads();
      count = sh.n;
    }
    for (uint32_t i = tid; i < count; i += BT) {
      const uint64_t p = sh.list[i];
      const float y = fkey_inv(pk_key(p));
      if (i >= kept)
        atomicAdd(&sh.fix, (unsigned long long)(long long)((exp((double)y - (double)now) - (double)term(y)) * 0x1p62));
      uint32_t rank = 0;
#pragma unroll 8
      for (uint32_t k = 0; k < count; ++k) rank += sh.list[k] > p;
      if (rank < n) sh.best[rank] = p;
    }
    kept = min(count, n);
  }
  __syncthreads();
  if (tid == 0) settle();
  uint64_t *out = tops + ((int64_t)row * parts + part) * n;
  if (tid < n) st_ag(out + tid, tid < kept ? sh.best[tid] : (uint64_t)0);
  sum = block_sum_f64(sum, sh.red);
  if (tid == 0) {
    ListSum *o = sums + (int64_t)row * parts + part;
    st_ag((uint64_t *)&o->sum, (uint64_t)__double_as_longlong(top_key > KEY_NEGINF ? sum : 0.0));
    st_ag((uint64_t *)&o->max, (uint64_t)__float_as_uint(top_key > KEY_NEGINF ? top : -INFINITY) | (uint64_t)(top_key >= KEY_POSINF) << 32);
  }
  store_wait();
  __syncthreads();
  if (tid == 0) sh.last = ticket_add(tick + blockIdx.y / a.beams) == a.beams * parts - 1;
  __syncthreads();
  if (!sh.last) return;
  if (tid == 0) st_ag(tick + blockIdx.y / a.beams, 0u);

  // ---- the join -----------------------------------------------------------------------------------------------------------
  const uint32_t total = a.beams * parts, entries = total * n;  // (lists, and what they hold)
  const ListSum *my = sums + (int64_t)r * total;
  const uint64_t *lists = tops + (int64_t)r * entries;
  uint64_t ahead[AHEAD];
#pragma unroll
  for (int j = 0; j < AHEAD; ++j) ahead[j] = j * BT + tid < entries ? ld_ag(lists + j * BT + tid) : 0;
  for (uint32_t i = tid; i < total; i += BT) {
    const uint64_t most = ld_ag((const uint64_t *)&my[i].max);
    sh.sums[i] = __longlong_as_double((long long)ld_ag((const uint64_t *)&my[i].sum));
    sh.maxs[i] = most >> 32 ? __uint_as_float(0x7FC00000u) : __uint_as_float((uint32_t)most);
  }
  const float my_score = lane < a.beams ? a.scores[(int64_t)r * a.beams + lane] : 0;
  __syncthreads();
  for (uint32_t b = wave; b < a.beams; b += BT / WAVE) {
    float bm = -INFINITY;
    bool bad = false;
    for (uint32_t i = lane; i < parts; i += WAVE) {
      const float y = sh.maxs[b * parts + i];
      bad = bad || y != y;
      bm = fmaxf(bm, y);
    }
    bm = wave_max_f32(bm);
    bad = ballot64(bad) != 0;
    double s = 0;
    for (uint32_t i = lane; i < parts; i += WAVE) {
      const double part_sum = sh.sums[b * parts + i];
      if (part_sum > 0) s += part_sum * exp((double)sh.maxs[b * parts + i] - (double)bm);
    }
    s = wave_sum_f64(s);
    const float score = __shfl(my_score, (int)b, WAVE);
    if (lane == 0) {
      const bool ok = !bad && bm > -INFINITY && isfinite(score);
      sh.base[b] = ok ? (double)bm : -INFINITY;  // (-inf: the beam gives nothing)
      sh.shift[b] = ok ? log(s) : 0.0;
      sh.score[b] = ok ? (double)score : 0.0;
    }
  }
  __syncthreads();
  auto value = [&](uint32_t i, uint64_t p, uint32_t &b) -> uint64_t {  // of entry i, of beam b; 0: none
    uint32_t rest;
    b = quotient(i, by_beam, rest);
    if (p == 0 || sh.base[b] == -INFINITY) return 0;
    return dkey(((double)fkey_inv(pk_key(p)) - sh.base[b]) - sh.shift[b] + sh.score[b]);
  };
  // a bound that n entries reach: the n-th largest of the threads' largest so far, by its upper 32 bits
  uint64_t lead = 0, val[AHEAD];
  uint32_t of[AHEAD];
#pragma unroll
  for (int j = 0; j < AHEAD; ++j) {
    val[j] = 0;
    if (j * BT < entries) val[j] = value(min(j * BT + tid, entries - 1), ahead[j], of[j]);
    lead = max(lead, val[j]);
  }
  const uint64_t from = max((uint64_t)block_kth_u32((uint32_t)(lead >> 32), n, (uint32_t *)sh.list) << 32, (uint64_t)1);
  if (tid == 0) sh.n = 0;
  __syncthreads();
  auto take = [&](uint64_t y, uint32_t b, uint64_t p) {
    if (y < from) return;
    const uint32_t at = atomicAdd(&sh.n, 1u);
    if (at < BL) {
      sh.list[at] = y;
      sh.sub[at] = (uint64_t)b << 32 | pk_id(p);
    }
  };
#pragma unroll
  for (int j = 0; j < AHEAD; ++j) take(val[j], of[j], ahead[j]);
#pragma unroll 4
  for (uint32_t i = AHEAD * BT + tid; i < entries; i += BT) {
    const uint64_t p = ld_ag(lists + i);
    uint32_t b;
    const uint64_t y = value(i, p, b);
    take(y, b, p);
  }
  __syncthreads();
  const uint32_t count = sh.n;
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
#pragma unroll 8
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
    for (uint32_t i = tid; i < entries; i += BT) {
      uint32_t b;
      const uint64_t p = ld_ag(lists + i), v = value(i, p, b);
      if (v == 0) continue;
      const uint64_t place = (uint64_t)b << 32 | pk_id(p);
      if ((v < lv || (v == lv && k > 0 && place > lp)) && (v > bv || (v == bv && place < bp))) {
        bv = v;
        bp = place;
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

// Workgroups of a row: a slice each while all of them run at once (four a CU), else as many as do: the device starts about 94
// workgroups a us, so that more rounds of short ones cost (64 x 8 rows of 151936: 65 us; with 8 a CU 74, with a slice each 129, with 2 a
// CU 82).
static uint32_t beam_parts(const gsk_beams &a, int cus) {
  const uint64_t slices = (a.vocab + BS - 1) / BS, rows = (uint64_t)a.requests * a.beams;
  const uint64_t most = std::max((uint64_t)4 * cus / std::max(rows, (uint64_t)1), (uint64_t)1);
  return (uint32_t)std::min(std::min(slices, most), (uint64_t)(LISTS / a.beams));
}

int64_t beam_work(const gsk_beams &a, int cus) {
  return (int64_t)a.requests * a.beams * beam_parts(a, cus) * (int64_t)(sizeof(ListSum) + a.n * sizeof(uint64_t));
}

hipError_t launch_beam(const gsk_beams &a, int cus, uint32_t *tick, uint32_t tickets, hipStream_t s) {
  const uint32_t parts = beam_parts(a, cus);
  // a launch takes a ticket per request, and 65535 rows at most
  const uint32_t most = std::min(tickets, 65535u / a.beams);
  auto go = [&](auto type, auto wide) {
    for (uint32_t r0 = 0; r0 < a.requests; r0 += most)
      hipLaunchKernelGGL((beam_kernel<type(), wide()>), dim3(parts, std::min(most, a.requests - r0) * a.beams), dim3(BT), 0, s, a, parts,
                         div_by(parts * a.n), tick, r0);
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
