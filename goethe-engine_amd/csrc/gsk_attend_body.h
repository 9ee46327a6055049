// The attention kernel of gsk_attend (gsk_attend.hip has the plan and the launches; one source per cache type instantiates it).
//
// A workgroup takes one part of one request's cached tokens, one head of the cache and one tile of up to 16 MT rows: a row is a
// (new token, query head of the group), so that every query head that reads a cached row shares its load. Its four waves take
// blocks of 64 tokens in turn, each with its own running maximum m, sum l and output O of every row (one pass: a tile's scores
// S, m' = max(m, S), p = 2^(S - m'), l = l 2^(m - m') + sum p, O = O 2^(m - m') + p V), joined through LDS at the end; the parts
// of a request are joined, in their order, by the last workgroup of a (request, head, tile) to end.
//
// Both products are 16x16x32 matrix instructions. S^T = K Q^T: a lane (c, g) = (lane % 16, lane / 16) holds eight elements of
// token c and of row c, and gets the scores of row c for tokens 4g .. 4g + 3 of each 16; O^T = V^T P^T over 32 tokens then takes
// those scores as they are, with the lane's eight of the 32 tokens numbered as S left them (4g + j of the first 16, 4g + j of
// the second). V is read as rows too, a lane eight elements (8c ...) of its eight tokens, and turned in registers: matrix
// instruction e of eight has element 8c + e as its row c. So nothing goes through LDS but the tokens' offsets (a lane finds one
// token's, a block ahead) and 8-bit scales. 8-bit elements are exact in 16 bits; their scales multiply S and p in fp32.
//
// The weights p are rounded to 16 bits for the second product (half a step each, 2^-8 relative in bfloat16, 2^-11 in float16;
// their sum l is of the unrounded ones). Over an 8-bit cache p times the token's scale is rounded, to bfloat16 whatever q's
// type: the products would leave float16's range.
#pragma once
#include "gsk_dev.h"
#include "gsk_int.h"

namespace gse {

constexpr int AT = 256, AW = AT / WAVE;
constexpr uint32_t AB = 64;  // tokens of a block

struct AttendArgs {
  gsk_cache c;
  gsk_attention a;
  uint32_t items, tiles, group, rows;  // rows: of a tile's scratch
  uint32_t *tick;
};

template <int KD>
struct AttendShared {
  static constexpr int VB = KD / 4, LD = 132;
  float o[AW][16][LD];       // a wave's O of 16 rows and 128 elements (padded by a bank row)
  float m[AW][16], l[AW][16];
  int64_t at[AW][AB];        // byte offsets of the block's tokens
  float ks[AW][AB], vs[AW][AB];
  int64_t red[AW];
  uint32_t item[4];          // request, part, parts, first item
  uint32_t last;
};

template <uint32_t T>
using Frag = std::conditional_t<T == GSK_F16, f16x8, bf16x8>;

template <uint32_t T>
__device__ __forceinline__ f32x4 mma(Frag<T> a, Frag<T> b, f32x4 c) {
  if constexpr (T == GSK_F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// Two 8-bit elements, bytes 2k and 2k + 1 of w, as T's pair.
template <uint32_t C, uint32_t T, int K>
__device__ __forceinline__ uint32_t widen(uint32_t w) {
  if constexpr (C == GSK_E4M3) {
    if constexpr (T == GSK_F16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, K != 0));
    else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, K != 0));
  } else {
    const float x = (float)((int32_t)(w << (K ? 8 : 24)) >> 24), y = (float)((int32_t)(w << (K ? 0 : 16)) >> 24);
    if constexpr (T == GSK_F16) return __builtin_bit_cast(uint32_t, f16x2{(_Float16)x, (_Float16)y});
    else return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)x, (__bf16)y});
  }
}

// Eight elements of a row as an operand of type T.
template <uint32_t C, uint32_t T>
__device__ __forceinline__ Frag<T> operand(const Raw8<C> &r) {
  if constexpr (type_is_8bit<C>) {
    uint4 w;
    w.x = widen<C, T, 0>(r.w[0]);
    w.y = widen<C, T, 1>(r.w[0]);
    w.z = widen<C, T, 0>(r.w[1]);
    w.w = widen<C, T, 1>(r.w[1]);
    return __builtin_bit_cast(Frag<T>, w);
  } else {
    return __builtin_bit_cast(Frag<T>, *(const uint4 *)r.w);
  }
}

// Element E of eight tokens' rows as an operand of type T.
template <uint32_t C, uint32_t T, int E>
__device__ __forceinline__ Frag<T> turned(const Raw8<C> (&v)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (type_is_8bit<C>) {
      const uint32_t a = v[2 * j].w[E / 4], b = v[2 * j + 1].w[E / 4];
      w[j] = widen<C, T, E & 1>(__builtin_amdgcn_perm(b, a, E & 2 ? 0x07030602u : 0x05010400u));
    } else {
      w[j] = __builtin_amdgcn_perm(v[2 * j + 1].w[E / 2], v[2 * j].w[E / 2], E & 1 ? 0x07060302u : 0x05040100u);
    }
  }
  return __builtin_bit_cast(Frag<T>, uint4{w[0], w[1], w[2], w[3]});
}

// The value over the lanes of the same lane % 16.
template <typename Op>
__device__ __forceinline__ float over_groups(float x, Op op) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = op(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return op(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// The factor of a part of maximum m and sum l in a whole of maximum top (NaN scores leave m at -inf and l NaN).
__device__ __forceinline__ float weight_of(float m, float l, float top) {
  return l == 0.0f ? 0.0f : m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - top);
}

struct Span {       // a request's rows and cached tokens
  int64_t begin;    // -1: nothing to write
  int32_t n, len;   // new tokens; cached ones, 0 where the request is not served
};
__device__ __forceinline__ Span span_of(const gsk_cache &c, const gsk_attention &a, uint32_t r) {
  const int64_t b = a.begin ? a.begin[r] : (int64_t)r, e = a.begin ? a.begin[r + 1] : (int64_t)r + 1, len = a.seq_len[r];
  const uint32_t st = a.status ? a.status[r] : 0;
  if (b < 0 || e > (int64_t)a.tokens || e <= b) return {-1, 0, 0};
  const bool ok = st == 0 && len >= e - b && len <= (int64_t)a.max_pages * c.page;
  return {b, (int32_t)(e - b), ok ? (int32_t)len : 0};
}

template <uint32_t Q, uint32_t C, int KD, int MT>
__global__ __launch_bounds__(AT) void attend_kernel(AttendArgs p) {
  using Sh = AttendShared<KD>;
  constexpr uint32_t VT = type_is_8bit<C> ? (uint32_t)GSK_BF16 : Q;  // type of the second product
  constexpr int VB = Sh::VB, SZ = type_size<C>;
  constexpr float INF = INFINITY;
  __shared__ Sh sh;
  const gsk_cache &c = p.c;
  const gsk_attention &a = p.a;
  const uint32_t tid = threadIdx.x, lane = lane_id(), lc = lane % 16, lg = lane / 16;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid / WAVE);
  // the tiles of an (item, head) run on one XCD (workgroups go round the eight of them)
  const uint32_t x8 = blockIdx.x / 8, unit = x8 / p.tiles * 8 + blockIdx.x % 8, tile = x8 % p.tiles;
  if (unit >= p.items * c.heads) return;
  const uint32_t item = unit / c.heads, head = unit - item * c.heads;

  // ---- which request and part this is ------------------------------------------------------------------------------------
  uint32_t r = item, part = 0, parts = 1, first_item = item, size = 0x7FFFFFC0u;
  if (p.items > a.requests) {
    // parts of one size, so that all requests' come to at most items: more of them than requests by items - requests
    int64_t total = 0;
    for (uint32_t i = tid; i < a.requests; i += AT) total += span_of(c, a, i).len;
    total = (int64_t)wave_sum_u64((uint64_t)total);
    if (lane == 0) sh.red[wave] = total;
    if (tid == 0) sh.item[0] = ~0u;
    __syncthreads();
    total = 0;
    for (int w = 0; w < AW; ++w) total += sh.red[w];
    const int64_t extra = p.items - a.requests;
    size = (uint32_t)max((total + extra - 1) / extra, (int64_t)(AB * AW));
    size = (size + AB - 1) / AB * AB;
    uint32_t before = 0;
    for (uint32_t i0 = 0; i0 < a.requests; i0 += AT) {
      const uint32_t i = i0 + tid;
      uint32_t n = 0;
      if (i < a.requests) n = max(((uint32_t)span_of(c, a, i).len + size - 1) / size, 1u);
      const uint32_t inc = wave_incl_scan_u32(n);
      __syncthreads();
      if (lane == WAVE - 1) sh.red[wave] = inc;
      __syncthreads();
      uint32_t at = before + inc - n;
      for (uint32_t w = 0; w < AW; ++w) {
        if (w < wave) at += (uint32_t)sh.red[w];
        before += (uint32_t)sh.red[w];
      }
      if (n > 0 && item >= at && item < at + n) {
        sh.item[0] = i;
        sh.item[1] = item - at;
        sh.item[2] = n;
        sh.item[3] = at;
      }
      if (before > item) break;
    }
    __syncthreads();
    r = __builtin_amdgcn_readfirstlane(sh.item[0]);
    if (r == ~0u) return;
    part = __builtin_amdgcn_readfirstlane(sh.item[1]);
    parts = __builtin_amdgcn_readfirstlane(sh.item[2]);
    first_item = __builtin_amdgcn_readfirstlane(sh.item[3]);
  }
  const Span sp = span_of(c, a, r);
  if (sp.begin < 0) return;
  const uint32_t rows = min((uint32_t)sp.n, a.max_new) * p.group, row0 = tile * 16 * MT;
  if (row0 >= rows) return;
  const uint32_t len = (uint32_t)sp.len, ctx = len >= (uint32_t)sp.n ? len - (uint32_t)sp.n : 0;
  const uint32_t last_new = (min(rows, row0 + 16 * MT) - 1) / p.group;
  const uint32_t k0 = part * size;  // (below 2^32: parts are at most the length's)
  uint32_t k1 = min(len, a.parent ? len : ctx + last_new + 1);
  if (k1 - min(k0, k1) > size) k1 = k0 + size;

  // ---- the rows -----------------------------------------------------------------------------------------------------------
  Frag<Q> q[MT][KD];
  uint32_t sees[MT];   // chains: the first cached token that the lane's row does not see
  uint64_t path[MT];   // trees: which new tokens it sees
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const uint32_t row = row0 + m * 16 + lc, i = min(row, rows - 1) / p.group, gi = min(row, rows - 1) - i * p.group;
    const char *at = (const char *)a.q + ((sp.begin + i) * a.q_token_stride + (int64_t)(head * p.group + gi) * a.q_head_stride) * 2;
#pragma unroll
    for (int k = 0; k < KD; ++k) {
      uint4 w = {0, 0, 0, 0};
      if (k * 32 + lg * 8 < c.dim) w = *(const uint4 *)(at + (k * 32 + lg * 8) * 2);
      q[m][k] = __builtin_bit_cast(Frag<Q>, w);
    }
    sees[m] = ctx + i + 1;
    path[m] = 0;
    if (a.parent) {
      int64_t at_ = sp.begin + i;
      for (;;) {  // (at most 64 steps: an ancestor is an earlier row)
        path[m] |= 1ull << (at_ - sp.begin);
        const int64_t up = a.parent[at_];
        if (up < sp.begin || up >= at_) break;
        at_ = up;
      }
    }
  }
  f32x4 acc[MT][VB][8];
  float mx[MT], l[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    mx[m] = -INF;
    l[m] = 0;
#pragma unroll
    for (int b = 0; b < VB; ++b)
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[m][b][e] = f32x4{0, 0, 0, 0};
  }

  // ---- the tokens ---------------------------------------------------------------------------------------------------------
  const float scale = a.scale * 1.44269504f;
  const char *keys = (const char *)c.keys + (int64_t)head * c.head_stride * SZ;
  const char *values = (const char *)c.values + (int64_t)head * c.head_stride * SZ;
  const int32_t *table = a.table + (int64_t)r * a.table_ld;
  uint32_t v_at[VB];  // (a lane past dim reads the row's start, into output elements that do not exist)
#pragma unroll
  for (int b = 0; b < VB; ++b) v_at[b] = b * 128 + lc * 8 < c.dim ? (b * 128 + lc * 8) * SZ : 0;

  auto page_of = [&](uint32_t t) -> uint32_t { return t < k1 ? (uint32_t)table[t / c.page] : ~0u; };
  uint64_t there = 0;  // the block's tokens that exist
  // A block's offsets and scales, from its tokens' pages, to LDS.
  auto place_block = [&](uint32_t t, uint32_t pg) {
    const bool ok = t < k1 && pg < c.pages;
    there = ballot64(ok);
    const uint32_t off = ok ? t % c.page : 0;
    if (!ok) pg = 0;
    sh.at[wave][lane] = ((int64_t)pg * c.page_stride + (int64_t)off * c.token_stride) * SZ;
    if constexpr (type_is_8bit<C>) {
      const int64_t s = (int64_t)pg * c.scale_page_stride + (int64_t)off * c.scale_token_stride + (int64_t)head * c.scale_head_stride;
      sh.ks[wave][lane] = c.key_scales[s];
      sh.vs[wave][lane] = c.value_scales[s];
    }
    __builtin_amdgcn_wave_barrier();
  };
  Raw8<C> kr[2][KD];
  auto load_keys = [&](uint32_t half) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const char *row = keys + sh.at[wave][half * 32 + s * 16 + lc];
#pragma unroll
      for (int k = 0; k < KD; ++k) {
        if (k * 32 >= (int)c.dim) continue;
        const bool in = k * 32 + lg * 8 < c.dim;
        kr[s][k] = load_raw8<C>(row + (in ? (k * 32 + lg * 8) * SZ : 0));
        if ((k + 1) * 32 > (int)c.dim && !in) kr[s][k] = Raw8<C>{};
      }
    }
  };

  uint32_t t0 = k0 + wave * AB;
  if (t0 < k1) {
    uint32_t pg = page_of(t0 + lane);
    place_block(t0 + lane, pg);
    load_keys(0);
    for (; t0 < k1; t0 += AW * AB) {
      const uint32_t next = t0 + AW * AB;
      pg = page_of(next + lane < next ? k1 : next + lane);
      const uint64_t now = there;
#pragma unroll
      for (uint32_t half = 0; half < 2; ++half) {
        const uint32_t t = t0 + half * 32;
        if (t >= k1) break;
        Raw8<C> vr[VB][8];
        float kscale[8], vscale[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t k = half * 32 + (j / 4) * 16 + lg * 4 + j % 4;
          const char *row = values + sh.at[wave][k];
#pragma unroll
          for (int b = 0; b < VB; ++b) vr[b][j] = load_raw8<C>(row + v_at[b]);
          if constexpr (type_is_8bit<C>) {
            kscale[j] = sh.ks[wave][k];
            vscale[j] = sh.vs[wave][k];
          }
        }
        f32x4 s[MT][2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
          for (int m = 0; m < MT; ++m) s[m][u] = f32x4{0, 0, 0, 0};
#pragma unroll
          for (int k = 0; k < KD; ++k) {
            if (k * 32 >= (int)c.dim) continue;
            const Frag<Q> kf = operand<C, Q>(kr[u][k]);
#pragma unroll
            for (int m = 0; m < MT; ++m) s[m][u] = mma<Q>(kf, q[m][k], s[m][u]);
          }
        }
        // the next tile's keys
        if (half == 0) {
          if (t + 32 < k1) load_keys(1);
        } else if (next < k1) {
          place_block(next + lane, pg);
          load_keys(0);
        }
        const uint32_t real = (uint32_t)(now >> (half * 32));
        const bool masked = real != ~0u || t + 32 > ctx;
        if (real != ~0u) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (!(real >> ((j / 4) * 16 + lg * 4 + j % 4) & 1))
#pragma unroll
              for (int b = 0; b < VB; ++b) vr[b][j] = Raw8<C>{};
        }
        Frag<VT> pf[MT];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          float z[8], top = -INF;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            z[j] = s[m][j / 4][j % 4] * scale;
            if constexpr (type_is_8bit<C>) z[j] *= kscale[j];
          }
          if (masked) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const uint32_t k = (j / 4) * 16 + lg * 4 + j % 4, at = t + k;
              bool see = real >> k & 1;
              if (at >= ctx) see = see && (a.parent ? (path[m] >> min(at - ctx, 63u) & 1) && at - ctx < 64 : at < sees[m]);
              if (!see) z[j] = -INF;
            }
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) top = fmaxf(top, z[j]);
          top = fmaxf(mx[m], over_groups(top, [](float x, float y) { return fmaxf(x, y); }));
          const float base = top == -INF ? 0.0f : top, f = __builtin_amdgcn_exp2f(mx[m] - base);
          mx[m] = top;
          float sum = 0;
          uint32_t w[4];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            z[j] = __builtin_amdgcn_exp2f(z[j] - base);
            sum += z[j];
            if constexpr (type_is_8bit<C>) z[j] *= vscale[j];
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if constexpr (VT == GSK_F16) w[j] = __builtin_bit_cast(uint32_t, f16x2{(_Float16)z[2 * j], (_Float16)z[2 * j + 1]});
            else w[j] = __builtin_bit_cast(uint32_t, bf16x2{(__bf16)z[2 * j], (__bf16)z[2 * j + 1]});
          }
          pf[m] = __builtin_bit_cast(Frag<VT>, uint4{w[0], w[1], w[2], w[3]});
          l[m] = l[m] * f + sum;
          if (ballot64(f != 1.0f)) {
#pragma unroll
            for (int b = 0; b < VB; ++b)
#pragma unroll
              for (int e = 0; e < 8; ++e) acc[m][b][e] *= f;
          }
        }
#pragma unroll
        for (int b = 0; b < VB; ++b) {
          auto step = [&]<int E>(std::integral_constant<int, E>) {
            const Frag<VT> vf = turned<C, VT, E>(vr[b]);
#pragma unroll
            for (int m = 0; m < MT; ++m) acc[m][b][E] = mma<VT>(vf, pf[m], acc[m][b][E]);
          };
          step(std::integral_constant<int, 0>{});
          step(std::integral_constant<int, 1>{});
          step(std::integral_constant<int, 2>{});
          step(std::integral_constant<int, 3>{});
          step(std::integral_constant<int, 4>{});
          step(std::integral_constant<int, 5>{});
          step(std::integral_constant<int, 6>{});
          step(std::integral_constant<int, 7>{});
        }
      }
    }
  }

  // ---- the waves' results joined ------------------------------------------------------------------------------------------
  // A thread has eight elements of one of 16 rows. A part's scratch: rows x dim of O, then rows x (m, l).
  float *work = (float *)a.work;
  const int64_t part_size = (int64_t)p.rows * (c.dim + 2);
  auto scratch = [&](uint32_t it) { return work + ((int64_t)(it * c.heads + head) * p.tiles + tile) * part_size; };
  const uint32_t tr = tid / 16, te = tid % 16 * 8;
  auto finish = [&](uint32_t row, uint32_t e, const float (&x)[8], float sum) {
    const uint32_t i = row / p.group, gi = row - i * p.group;
    const float inv = sum > 0 ? 1.0f / sum : 0.0f;
    float y[8];
#pragma unroll
    for (int d = 0; d < 8; ++d) y[d] = sum == 0 ? 0.0f : sum > 0 ? x[d] * inv : x[d] / sum;
    store_raw8<Q>((char *)a.out + (((sp.begin + i) * a.heads + head * p.group + gi) * (int64_t)c.dim + e) * 2, from_f32<Q>(y));
  };
#pragma unroll 1
  for (int m = 0; m < MT; ++m) {
    if (row0 + m * 16 >= rows) break;
#pragma unroll 1
    for (int b = 0; b < VB; ++b) {
      if (m || b) __syncthreads();
      // (the accumulators are picked with constant indexes)
#pragma unroll
      for (int mm = 0; mm < MT; ++mm) {
#pragma unroll
        for (int bb = 0; bb < VB; ++bb) {
          if (mm != m || bb != b) continue;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float *o = &sh.o[wave][lc][8 * (lg * 4 + i)];
            *(f32x4 *)o = f32x4{acc[mm][bb][0][i], acc[mm][bb][1][i], acc[mm][bb][2][i], acc[mm][bb][3][i]};
            *(f32x4 *)(o + 4) = f32x4{acc[mm][bb][4][i], acc[mm][bb][5][i], acc[mm][bb][6][i], acc[mm][bb][7][i]};
          }
          const float sum = over_groups(l[mm], [](float x, float y) { return x + y; });
          if (lg == 0) {
            sh.m[wave][lc] = mx[mm];
            sh.l[wave][lc] = sum;
          }
        }
      }
      __syncthreads();
      const uint32_t row = row0 + m * 16 + tr, e = b * 128 + te;
      if (row >= rows || e >= c.dim) continue;
      float top = -INF, sum = 0, x[8] = {};
#pragma unroll
      for (int w = 0; w < AW; ++w) top = fmaxf(top, sh.m[w][tr]);
#pragma unroll
      for (int w = 0; w < AW; ++w) {
        const float f = weight_of(sh.m[w][tr], sh.l[w][tr], top);
        if (f == 0.0f) continue;
        sum += f * sh.l[w][tr];
#pragma unroll
        for (int d = 0; d < 8; ++d) x[d] += f * sh.o[w][tr][te + d];
      }
      if (parts == 1) {
        finish(row, e, x, sum);
        continue;
      }
      float *o = scratch(item) + (int64_t)(row - row0) * c.dim + e;
#pragma unroll
      for (int d = 0; d < 8; d += 2) st_ag((uint64_t *)(o + d), (uint64_t)__float_as_uint(x[d]) | (uint64_t)__float_as_uint(x[d + 1]) << 32);
      if (e == 0)
        st_ag((uint64_t *)(scratch(item) + (int64_t)p.rows * c.dim + 2 * (row - row0)),
              (uint64_t)__float_as_uint(top) | (uint64_t)__float_as_uint(sum) << 32);
    }
  }
  if (parts == 1) return;

  // ---- the parts joined ---------------------------------------------------------------------------------------------------
  store_wait();
  __syncthreads();
  uint32_t *tick = p.tick + ((int64_t)r * c.heads + head) * p.tiles + tile;
  if (tid == 0) sh.last = ticket_add(tick) == parts - 1;
  __syncthreads();
  if (!sh.last) return;
  if (tid == 0) st_ag(tick, 0u);
  for (uint32_t i = tr; i < min(rows - row0, 16u * MT); i += 16) {
    float top = -INF;
    for (uint32_t s = 0; s < parts; ++s)
      top = fmaxf(top, __uint_as_float((uint32_t)ld_ag((const uint64_t *)(scratch(first_item + s) + (int64_t)p.rows * c.dim + 2 * i))));
#pragma unroll
    for (int b = 0; b < VB; ++b) {
      const uint32_t e = b * 128 + te;
      if (e >= c.dim) continue;
      float sum = 0, x[8] = {};
      for (uint32_t s = 0; s < parts; ++s) {
        const float *o = scratch(first_item + s);
        const uint64_t ml = ld_ag((const uint64_t *)(o + (int64_t)p.rows * c.dim + 2 * i));
        uint64_t w[4];
#pragma unroll
        for (int d = 0; d < 4; ++d) w[d] = ld_ag((const uint64_t *)(o + (int64_t)i * c.dim + e + 2 * d));
        const float part_l = __uint_as_float((uint32_t)(ml >> 32)), f = weight_of(__uint_as_float((uint32_t)ml), part_l, top);
        if (f == 0.0f) continue;
        sum += f * part_l;
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          x[2 * d] += f * __uint_as_float((uint32_t)w[d]);
          x[2 * d + 1] += f * __uint_as_float((uint32_t)(w[d] >> 32));
        }
      }
      finish(row0 + i, e, x, sum);
    }
  }
}

template <uint32_t Q, uint32_t C>
void launch_attend_types(const AttendArgs &p, int mt, dim3 grid, hipStream_t s) {
  auto go = [&](auto kd, auto m) { hipLaunchKernelGGL((attend_kernel<Q, C, kd(), m()>), grid, dim3(AT), 0, s, p); };
  auto by = [&](auto kd) {
    if (mt == 1) go(kd, std::integral_constant<int, 1>{});
    else if (mt == 2) go(kd, std::integral_constant<int, 2>{});
    else if constexpr (kd() == 4) go(kd, std::integral_constant<int, 4>{});
  };
  if (p.c.dim <= 128) by(std::integral_constant<int, 4>{});
  else by(std::integral_constant<int, 8>{});
}

// (q and cache types)
void launch_attend_bf16(const AttendArgs &p, int mt, dim3 grid, hipStream_t s);
void launch_attend_f16(const AttendArgs &p, int mt, dim3 grid, hipStream_t s);
void launch_attend_bf16_e4m3(const AttendArgs &p, int mt, dim3 grid, hipStream_t s);
void launch_attend_f16_e4m3(const AttendArgs &p, int mt, dim3 grid, hipStream_t s);
void launch_attend_bf16_i8(const AttendArgs &p, int mt, dim3 grid, hipStream_t s);
void launch_attend_f16_i8(const AttendArgs &p, int mt, dim3 grid, hipStream_t s);

}  // namespace gse
