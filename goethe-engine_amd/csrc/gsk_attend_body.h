// The attention kernel of gsk_attend (gsk_attend.hip has the plan and the launches; one source per cache type instantiates it).
//
// The work is a line of blocks of cached tokens: each request's tokens once for every tile of up to 16 MT of its rows, request after
// request. It is cut into equal shares of whole blocks, as many as workgroups run at once (at most p.items): a workgroup takes one share
// and one head of the cache, and works on the tiles (or parts of them) in its share in turn, so that requests with many new tokens and
// with one, in one call, take what they need (24 requests of up to 400 new tokens, 260 us; 765 with workgroups for each tile of every
// request). A row is a (new token, query head of the group), so that every query head
// that reads a cached row shares its load. The four waves take blocks of 32 tokens in turn, each with its own running maximum m,
// sum l and output O of every row (one pass: a block's scores S, m' = max(m, S), p = 2^(S - m'), l = l 2^(m - m') + sum p, O =
// O 2^(m - m') + p V), joined through LDS at the end; the parts of a tile are joined, in their order, by the last workgroup
// of a (request, tile, head) to end.
//
// Both products are 16x16x32 matrix instructions. S^T = K Q^T: a lane (c, g) = (lane % 16, lane / 16) holds eight elements of
// token c and of row c, and gets the scores of row c for tokens 4g .. 4g + 3 of each 16; O^T = V^T P^T over 32 tokens then takes
// those scores as they are, with the lane's eight of the 32 tokens numbered as S left them (4g + j of the first 16, 4g + j of
// the second). V is read as rows too, a lane eight elements (8c ...) of its eight tokens, and turned in registers: matrix
// instruction e of eight has element 8c + e as its row c. So nothing goes through LDS but the tokens' offsets (a lane finds one
// token's, a block ahead) and 8-bit scales. 8-bit elements are exact in 16 bits; their scales multiply S and p in fp32.
//
// The weights p (up to 2^8: the maximum lags) go into the second product as two 16-bit numbers, so that results are off by little
// more than their own rounding (with one, half a step of each weight, bfloat16's rms error was up to a seventh more). Over a 16-bit
// cache a weight is cut off and its rest rounded, off by 2^-15 of it in bfloat16 and 2^-20 in float16: both above 0, so that an
// infinite value times them is the same infinity (float16: at weights down to 2^-20 of the largest; below, it may become NaN). Over
// an 8-bit cache, whose values are finite or NaN, a weight is p times the token's scale, which may leave float16's range: two
// bfloat16 numbers, rounded and the rest (2^-16), whatever q's type.
//
// Bound: memory, by how the rows lie and by how evenly the workgroups of a CU get on. 128 requests of up to 16384 tokens of 8 heads of
// 128 8-bit elements (2.79 GB, 2.83 read by the counters), 8 rows a head: 534 us, 5.2 TB/s; with the heads ahead of a page's tokens 481 us,
// 5.8 TB/s (one head's tokens are then one stretch of memory). 96 trees of 9 new tokens over up to 4096 tokens of 16 bits (1.03 GB, 36
// rows a head): 249 us, 4.1 TB/s; of one new token 230. One request of 8192 tokens (34 MB): 20 to 22 us, a chain: lengths and table 4 us,
// two blocks a wave 6, the waves' join 2, the ticket 1, the parts' join 6. More shares than workgroups that run at once, so that those
// that end early take another, cost as the heads of an item fall apart (trees 285 us with two, 323 with four; batch 605, 653).
#pragma once
#include "gsk_dev.h"
#include "gsk_int.h"

namespace gse {

constexpr int AT = 256, AW = AT / WAVE;
constexpr uint32_t AB = 32;  // tokens of a block
// Blocks of a share, at least, and what a request's turn costs besides its tokens, in blocks (a share's requests count it). One request
// of up to 2048 and 8192 tokens: 15.4 and 22.1 us; with shares of 4 blocks 15.5 and 27.8 (twice the parts to join), of 16 18.0 and
// 20.2. 16 trees of up to 4096 tokens: 59.0 us, with a turn of 4 65.5, of 14 60.7.
constexpr uint32_t SHARE_MIN = 8, TURN = 8;
constexpr uint32_t FOUR_MIN = 32;   // blocks of a share, at least, where the waves take four heads

struct AttendArgs {
  gsk_cache c;
  gsk_attention a;
  uint32_t items, group, rows;  // shares, at most; query heads of a head; rows of a tile's scratch
  uint32_t *tick;
  uint32_t items4;  // shares where the waves take four heads (0: never)
};

template <int KD, int MT>
struct AttendShared {
  static constexpr int VB = (KD + 3) / 4, LD = 132;
  union {
    struct {                       // the tokens' loop
      uint4 q[MT == 1 ? AW : MT][16][KD * 4 + 1]; // the rows' operands (a piece of padding: the rows' pieces lie in different banks)
      int64_t at[AW][AB];          // byte offsets of the block's tokens
      float scale[AW][2][AB];      // and their keys' and values' scales
    };
    struct {                       // the joins
      float o[AW][16][LD];         // a wave's O of 16 rows and 128 elements
      float m[AW][16], l[AW][16];
    };
  };
  uint32_t last, bad[AW];
};

// Workgroups of a CU at once (what their registers allow; of MT = 1, four a CU left the loop spills and were slower).
constexpr int attend_resident(int kd, int mt) { return kd > 4 ? 1 : mt > 1 ? 2 : 3; }

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

// Makes finite numbers of the NaNs and infinities of eight elements (their exponents' upper bit cleared), if `on`; nonzero if
// there are any.
template <uint32_t C>
__device__ __forceinline__ uint32_t tame(Raw8<C> &r, bool on) {
  constexpr uint32_t ALL = C == GSK_BF16 ? 0x7F807F80u : C == GSK_F16 ? 0x7C007C00u : 0x7F7F7F7Fu;
  constexpr uint32_t ONE = C == GSK_BF16 ? 0x00800080u : C == GSK_F16 ? 0x04000400u : 0x01010101u;
  const uint32_t top = on ? type_is_8bit<C> ? 0x80808080u : 0x80008000u : 0u;
  uint32_t any = 0;
#pragma unroll
  for (int i = 0; C != GSK_I8 && i < Raw8<C>::N; ++i) {
    const uint32_t bad = ((r.w[i] & ALL) + ONE) & top;  // (8 bits: the one magnitude that is no number)
    r.w[i] &= ~(bad >> 1);
    any |= bad;
  }
  return any;
}

// The value over the lanes of the same lane % 16.
template <typename Op>
__device__ __forceinline__ float over_groups(float x, Op op) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = op(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return op(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// The factor of a part of maximum m and sum l in a whole of maximum top (NaN scores leave m at -inf and l NaN). A part that saw
// nothing has l 0 and is left out; one whose factor is 0 is not: its NaNs and infinities count.
__device__ __forceinline__ float weight_of(float m, float l, float top) {
  return l == 0.0f ? 0.0f : m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - top);
}

struct Raw {        // a request's numbers as they are
  int32_t begin, end, len;
  uint32_t status;
};
__device__ __forceinline__ Raw raw_of(const gsk_attention &a, uint32_t r) {
  Raw x{(int32_t)r, (int32_t)r + 1, a.seq_len[r], 0};
  if (a.begin) x.begin = a.begin[r], x.end = a.begin[r + 1];
  if (a.status) x.status = a.status[r];
  return x;
}
struct Span {       // a request's rows and cached tokens
  int32_t begin;    // -1: nothing to write
  int32_t n, len;   // new tokens; cached ones, 0 where the request is not served
};
__device__ __forceinline__ Span span_of(const gsk_cache &c, const gsk_attention &a, Raw x) {
  if (x.begin < 0 || x.end < 0 || (uint32_t)x.end > a.tokens || x.end <= x.begin) return {-1, 0, 0};
  const int32_t n = x.end - x.begin;
  const bool ok = x.status == 0 && x.len >= n && (int64_t)x.len <= (int64_t)a.max_pages * c.page;
  return {x.begin, n, ok ? x.len : 0};
}
// A request's turns, one for each tile of its rows (of 16 MT), and the blocks that a turn counts.
struct Turns {
  uint32_t n, blocks;
};
template <int MT>
__device__ __forceinline__ Turns turns_of(const gsk_attention &a, uint32_t group, Span x) {
  if (x.begin < 0) return {0, 0};
  return {(min((uint32_t)x.n, a.max_new) * group + 16 * MT - 1) / (16 * MT), TURN + max(((uint32_t)x.len + AB - 1) / AB, 1u)};
}

template <uint32_t Q, uint32_t C, int KD, int MT>
__global__ __launch_bounds__(AT, attend_resident(KD, MT)) void attend_kernel(AttendArgs p) {
  using Sh = AttendShared<KD, MT>;
  constexpr uint32_t VT = type_is_8bit<C> ? (uint32_t)GSK_BF16 : Q;  // type of the second product
  constexpr int VB = Sh::VB, SZ = type_size<C>;
  constexpr float INF = INFINITY;
  // 16 bits: a weight times MORE goes into the second product, cut off and the rest, which then is above 0 (an infinite value stays one)
  constexpr float MORE = type_is_8bit<C> ? 1.0f : VT == GSK_F16 ? 1.0f + 0x1p-12f : 1.0f + 0x1p-17f;
  __shared__ Sh sh;
  const gsk_cache &c = p.c;
  const gsk_attention &a = p.a;
  const uint32_t tid = threadIdx.x, lane = lane_id(), lc = lane % 16, lg = lane / 16;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid / WAVE);
  // ---- the share ----------------------------------------------------------------------------------------------------------
  // Every wave for itself, a lane one request or, where there are more than lanes, four at a time: a tile's blocks, one at least if
  // there are rows to write, after TURN that stand for its turn. The shares are of one size, the first ones a block more.
  const int per = a.requests <= WAVE ? 1 : 4;
  Span own[4];
  uint32_t u[4] = {};
  auto take = [&](uint32_t i0) {  // returns the lane's blocks
    uint32_t n = 0;
    Raw raw[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < per) raw[k] = raw_of(a, min(i0 + lane * per + k, a.requests - 1));
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (k >= per) continue;
      own[k] = span_of(c, a, raw[k]);
      const Turns w = turns_of<MT>(a, p.group, own[k]);
      u[k] = i0 + lane * per + k < a.requests ? w.n * w.blocks : 0;
      n += u[k];
    }
    return n;
  };
  uint32_t mine = take(0), total = mine;  // (below 2^32 by the host's check)
  for (uint32_t i0 = 4 * WAVE; i0 < a.requests; i0 += 4 * WAVE) total += take(i0);
  total = wave_sum_u32(total);
  // Four heads: where a token's heads lie together and the host finds it worth it (attend_plan), with tokens enough, a wave takes
  // every block of the share for one of four heads, and nothing is joined between waves.
  const bool four = MT == 1 && p.items4 && total >= p.items4 * FOUR_MIN;
  const uint32_t shares = four ? p.items4 : min(max(total / SHARE_MIN, 1u), p.items);
  // The heads of an item run on one XCD (workgroups go round the eight of them): a token's heads lie together.
  const uint32_t x8 = blockIdx.x / 8, each = four ? c.heads / AW : c.heads, x = x8 % each;
  const uint32_t item = x8 / each * 8 + blockIdx.x % 8, head0 = x * (four ? AW : 1);
  const uint32_t head = four ? head0 + wave : head0, heads_here = four ? AW : 1;
  if (item >= shares) return;
  const uint32_t share = total / shares, longer = total - share * shares;
  auto first_of = [&](uint32_t w) { return w * share + min(w, longer); };
  auto share_of = [&](uint32_t block) {
    const uint32_t border = longer * (share + 1);
    return block < border ? block / (share + 1) : longer + (block - border) / share;
  };
  uint32_t pos = first_of(item), start = 0;  // the share's first block; the first block of request r
  const uint32_t stop = first_of(item + 1);
  const uint32_t share0 = pos, quarter = max((stop - pos) / 4, 1u) * AB;
  if (pos >= stop) return;  // (nothing to write at all)
  uint32_t r = 0;
  Span sp;
  for (uint32_t i0 = 0;; i0 += 4 * WAVE) {
    if (a.requests > 4 * WAVE) mine = take(i0);
    const uint32_t inc = wave_incl_scan_u32(mine);
    const uint64_t past = ballot64(start + inc > pos);
    if (!past) {
      start += lane63(inc);
      continue;
    }
    const int at = __builtin_ctzll(past);
    start += __builtin_amdgcn_readlane(inc - mine, at);
    r = i0 + at * per;
    bool found = false;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (found || k >= per) continue;
      sp.begin = __builtin_amdgcn_readlane(own[k].begin, at);
      sp.n = __builtin_amdgcn_readlane(own[k].n, at);
      sp.len = __builtin_amdgcn_readlane(own[k].len, at);
      const uint32_t n = __builtin_amdgcn_readlane(u[k], at);
      found = k + 1 >= per || start + n > pos;
      if (!found) {
        start += n;
        ++r;
      }
    }
    break;
  }
  start = __builtin_amdgcn_readfirstlane(start);
  r = __builtin_amdgcn_readfirstlane(r);
  Turns turns = turns_of<MT>(a, p.group, sp);
  uint32_t tile = turns.n ? (pos - start) / turns.blocks : 0;
  start += tile * turns.blocks;

  Raw ahead;
  auto next = [&] {  // the request's next tile, or the next request
    if (++tile < turns.n) return;
    tile = 0;
    sp = span_of(c, a, ahead);
    turns = turns_of<MT>(a, p.group, sp);
    ++r;
  };
  for (;; next()) {
  if (pos >= stop) break;
  ahead = raw_of(a, min(r + 1, a.requests - 1));  // (the next request's, for the next turn)
  if (sp.begin < 0) continue;
  const uint32_t first = start + TURN, end = start + turns.blocks, from = max(pos, first);  // the request's blocks
  start = end;
  pos = min(stop, end);
  if (from >= pos) continue;  // (the share ends within its turn)
  const uint32_t k0 = (from - first) * AB, k_end = (pos - first) * AB;
  const uint32_t first_item = from == first ? item : share_of(first), parts = (end <= stop ? item : share_of(end - 1)) - first_item + 1;
  const uint32_t rows = min((uint32_t)sp.n, a.max_new) * p.group, row0 = tile * 16 * MT;
  const uint32_t len = (uint32_t)sp.len, ctx = len >= (uint32_t)sp.n ? len - (uint32_t)sp.n : 0;
  const uint32_t last_new = (min(rows, row0 + 16 * MT) - 1) / p.group;
  const uint32_t k1 = min(k_end, a.parent ? len : min(len, ctx + last_new + 1));

  // ---- the rows -----------------------------------------------------------------------------------------------------------
  const uint32_t sign = a.scale < 0 ? 0x80008000u : 0;  // (the scale's own, so that the largest score is the largest product)
  constexpr int QN = ((MT == 1 ? AW : MT) * 16 * KD * 4 + AT - 1) / AT;
  uint4 rows_q[QN];  // (to LDS once the first block's loads are on their way)
#pragma unroll
  for (int j = 0; j < QN; ++j) {
    const uint32_t at_q = j * AT + tid, w = at_q / (KD * 4), e = at_q % (KD * 4);
    const uint32_t row = min(row0 + (four ? w % 16 : w), rows - 1), n = row / p.group, h = head0 + (four ? w / 16 : 0);
    rows_q[j] = uint4{0, 0, 0, 0};
    if (w < (four ? AW : MT) * 16 && e * 8 < c.dim)
      rows_q[j] = *(const uint4 *)((const char *)a.q + ((int64_t)(sp.begin + n) * a.q_token_stride +
                                                        (int64_t)(h * p.group + row - n * p.group) * a.q_head_stride + e * 8) * 2);
  }
  auto q_of = [&](int m, int k) { return __builtin_bit_cast(Frag<Q>, sh.q[four ? wave : m][lc][k * 4 + lg]); };
  uint32_t sees[MT];   // chains: the first cached token that the lane's row does not see
  uint64_t path[MT];   // trees: which new tokens it sees
  const int32_t parent = a.parent ? a.parent[sp.begin + (int32_t)min(lane, (uint32_t)sp.n - 1)] : 0;  // of new token `lane`
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const uint32_t i = min(row0 + m * 16 + lc, rows - 1) / p.group;
    sees[m] = ctx + i + 1;
    path[m] = 0;
    if (a.parent) {  // (uniform; at most 64 steps: an ancestor is an earlier row)
      uint32_t node = i;
      bool on = true;
      while (ballot64(on)) {
        if (on) path[m] |= 1ull << node;
        const int32_t up = __shfl(parent, (int)node, WAVE) - sp.begin;
        on = on && up >= 0 && (uint32_t)up < node;
        if (on) node = (uint32_t)up;
      }
    }
  }
  f32x4 acc[MT][VB][8];
  // What the running maximum has added to it. Over float16 the weights are 2^7 as large, up to 2^15, so that those below 2^-14 of the
  // largest, whose steps are 2^-24, count to 2^-32 of it (a long tail behind one token that outweighs each of them). In bfloat16 the
  // weights of all tokens add up to less than 1/2, so that no sum of values, or scale times weight, leaves fp32's range (what is lost
  // at its other end is below 2^-126 times 2^9 and the tokens).
  const float drop = VT == GSK_F16 ? -7.0f : (float)(9 + 32 - __builtin_clz(len | 1));
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
  // The loads of a block are in one straight line, the next block's keys and the offsets of the one after ahead of what is worked
  // on: a load behind a branch would make every later wait one for all loads. Tokens that do not exist read slot 0 and are
  // masked. Lanes l and l + 32 find the same token.
  const float scale = fabsf(a.scale) * 1.44269504f;
  const int32_t *table = a.table + (int64_t)r * a.table_ld;
  const uint32_t hop = four ? AB : AW * AB, pages_on = hop / c.page, tokens_on = hop % c.page;  // to the wave's next block
  const uint32_t l32 = lane % 32;
  uint32_t t = k0 + (four ? 0 : wave * AB);
  uint32_t pi = (t + l32) / c.page, off = (t + l32) % c.page;  // the lane's token of the next block
  const uint32_t last_page = (max(k1, 1u) - 1) / c.page;
  auto next_page = [&] { return (uint32_t)table[min(pi, last_page)]; };
  uint32_t there = 0;  // the tokens of the block that sh.at has
  uint32_t bad = 0;    // NaNs or infinities among values that some rows do not see
  float scale_of = 0;  // 8 bits: the token's, of its key in the lower lanes and of its value in the upper ones
  const float *scales = lane < 32 ? c.key_scales : c.value_scales;
  auto place_block = [&](uint32_t t, uint32_t pg) {  // the offsets of a block to LDS, from its tokens' pages
    const bool ok = t < k1 && pg < c.pages;
    there = (uint32_t)ballot64(ok);
    const uint32_t o = ok ? off : 0;
    if (!ok) pg = 0;
    sh.at[wave][l32] = ((int64_t)pg * c.page_stride + (int64_t)o * c.token_stride) * SZ;
    if constexpr (type_is_8bit<C>)
      scale_of = scales[(int64_t)pg * c.scale_page_stride + (int64_t)o * c.scale_token_stride + (int64_t)head * c.scale_head_stride];
    pi += pages_on;
    off += tokens_on;
    if (off >= c.page) off -= c.page, ++pi;
    __builtin_amdgcn_wave_barrier();
  };
  // A lane's part of a row: eight elements at 32k + 8g of a key, at 128b + 8c of a value. Past dim it reads what is there anyway:
  // keys are zeroed then, values go into output elements that do not exist. WHOLE: the key chunks that are never past it.
  constexpr int WHOLE = KD == 8 ? 4 : KD >= 3 ? KD - 1 : 0;
  const char *keys = (const char *)c.keys + ((int64_t)head * c.head_stride + lg * 8) * SZ;
  const char *values = (const char *)c.values + (int64_t)head * c.head_stride * SZ + (lc * 8 < c.dim ? lc * 8 * SZ : 0);
  int32_t k_at[KD - WHOLE], v_at = 0;
#pragma unroll
  for (int k = WHOLE; k < KD; ++k) k_at[k - WHOLE] = (k * 32 + lg * 8 < c.dim ? k * 32 : -(int)lg * 8) * SZ;
  if (VB > 1) v_at = (128 + lc * 8 < c.dim ? 128 : -(int)lc * 8) * SZ;
  const bool whole = c.dim == KD * 32;
  Raw8<C> kr[2][KD];
  auto load_keys = [&] {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const char *row = keys + sh.at[wave][s * 16 + lc];
#pragma unroll
      for (int k = 0; k < KD; ++k) kr[s][k] = load_raw8<C>(k < WHOLE ? row + k * 32 * SZ : row + k_at[k < WHOLE ? 0 : k - WHOLE]);
    }
  };

  if (t < k1) {
    place_block(t + l32, next_page());
    load_keys();
  }
#pragma unroll
  for (int j = 0; j < QN; ++j) {
    const uint32_t at_q = j * AT + tid, w = at_q / (KD * 4);
    uint4 v = rows_q[j];
    v.x ^= sign, v.y ^= sign, v.z ^= sign, v.w ^= sign;
    if (w < (four ? AW : MT) * 16) sh.q[w / 16][w % 16][at_q % (KD * 4)] = v;
  }
  __syncthreads();
  if (t < k1) {
    for (; t < k1; t += hop) {
      if constexpr (type_is_8bit<C>) {
        // A wave that has done more of its share gives way. The older workgroup of a CU goes first otherwise, and the heads of an item,
        // which read one stretch of memory, fall apart: 128 requests up to 16384 tokens 554 -> 533 us (the workgroups' ends lay
        // between 290 and 560). Over 16-bit rows, where the waves issue less, it changed nothing.
        const uint32_t done = t - k0 + (from - share0) * AB;
        if (done < quarter) __builtin_amdgcn_s_setprio(3);
        else if (done < 2 * quarter) __builtin_amdgcn_s_setprio(2);
        else if (done < 3 * quarter) __builtin_amdgcn_s_setprio(1);
        else __builtin_amdgcn_s_setprio(0);
      }
      const uint32_t page = next_page(), real = there;
      if constexpr (type_is_8bit<C>) sh.scale[wave][lane / 32][l32] = lane < 32 ? scale_of * scale : scale_of;
      Raw8<C> vr[VB][8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const char *row = values + sh.at[wave][(j / 4) * 16 + lg * 4 + j % 4];
#pragma unroll
        for (int b = 0; b < VB; ++b) vr[b][j] = load_raw8<C>(b ? row + v_at : row);
      }
      if (!whole) {  // (what a lane past dim has read)
#pragma unroll
        for (int k = WHOLE; k < KD; ++k)
          if (k * 32 + lg * 8 >= c.dim) kr[0][k] = kr[1][k] = Raw8<C>{};
      }
      f32x4 s[MT][2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int m = 0; m < MT; ++m) s[m][u] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < KD; ++k) {
          const Frag<Q> kf = operand<C, Q>(kr[u][k]);
#pragma unroll
          for (int m = 0; m < MT; ++m) s[m][u] = mma<Q>(kf, q_of(m, k), s[m][u]);
        }
      }
      place_block(t + hop + l32, page);
      load_keys();
      f32x4 kscale[2], vscale[2];
      if constexpr (type_is_8bit<C>) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          kscale[u] = *(const f32x4 *)&sh.scale[wave][0][u * 16 + lg * 4];
          vscale[u] = *(const f32x4 *)&sh.scale[wave][1][u * 16 + lg * 4];
        }
      }
      const bool masked = real != ~0u || t + 32 > ctx;
      Frag<VT> pf[MT], rest[MT];  // (what the first rounding leaves)
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        float z[8], top = -INF;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          z[j] = s[m][j / 4][j % 4];
          if constexpr (type_is_8bit<C>) z[j] *= kscale[j / 4][j % 4];
        }
        if (masked) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const uint32_t k = (j / 4) * 16 + lg * 4 + j % 4, at = t + k, d = at - ctx;  // (past ctx: the new token's index)
            const uint32_t in_new = a.parent ? (uint32_t)(path[m] >> (d & 63)) & (uint32_t)(d < 64) : (uint32_t)(at < sees[m]);
            const uint32_t see = (real >> k) & ((uint32_t)(at < ctx) | in_new) & 1;
            if constexpr (type_is_8bit<C>) z[j] = __builtin_fmaf(vscale[j / 4][j % 4], 0.0f, z[j]);  // (a value's NaN, at any weight)
            z[j] = see ? z[j] : -INF;
          }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) top = fmaxf(top, z[j]);
        top = over_groups(top, [](float x, float y) { return fmaxf(x, y); });
        if constexpr (!type_is_8bit<C>) top = top == -INF ? -INF : top * scale;  // (a scale of 0)
        // The maximum follows once it is 2^8 behind: the weights are up to that, and what it saves is the output's rescaling.
        top += drop;
        if (ballot64(top > mx[m] + 8.0f)) {
          top = top > mx[m] + 8.0f ? top : mx[m];  // (a row's own: what others see does not change it)
          const float f = __builtin_amdgcn_exp2f(mx[m] - (top == -INF ? 0.0f : top));
          mx[m] = top;
          l[m] *= f;
#pragma unroll
          for (int b = 0; b < VB; ++b)
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[m][b][e] *= f;
        }
        const float base = mx[m] == -INF ? 0.0f : mx[m];
        uint32_t w[4], d[4];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if constexpr (type_is_8bit<C>) z[j] = __builtin_amdgcn_exp2f(z[j] - base);
          else z[j] = __builtin_amdgcn_exp2f(z[j] == -INF ? -INF : __builtin_fmaf(z[j], scale, -base));
          l[m] += z[j];
          if constexpr (type_is_8bit<C>) {
            const float v = z[j] * vscale[j / 4][j % 4];
            z[j] = masked && z[j] == 0.0f ? 0.0f : v;  // (the scale of a token that is not seen may be NaN)
          }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if constexpr (VT == GSK_F16) {
            const f16x2 h = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_pkrtz(z[2 * j], z[2 * j + 1]));
            w[j] = __builtin_bit_cast(uint32_t, h);
            d[j] = __builtin_bit_cast(uint32_t, f16x2{(_Float16)__builtin_fmaf(z[2 * j], MORE, -(float)h.x),
                                                      (_Float16)__builtin_fmaf(z[2 * j + 1], MORE, -(float)h.y)});
          } else if constexpr (type_is_8bit<C>) {
            w[j] = __builtin_bit_cast(uint32_t, bf16x2{(__bf16)z[2 * j], (__bf16)z[2 * j + 1]});
            const float x = __uint_as_float(w[j] << 16), y = __uint_as_float(w[j] & 0xFFFF0000u);
            d[j] = __builtin_bit_cast(uint32_t, bf16x2{(__bf16)(z[2 * j] - x), (__bf16)(z[2 * j + 1] - y)});
          } else {
            const uint32_t x = __float_as_uint(z[2 * j]), y = __float_as_uint(z[2 * j + 1]);
            w[j] = __builtin_amdgcn_perm(y, x, 0x07060302u);
            d[j] = __builtin_bit_cast(uint32_t, bf16x2{(__bf16)__builtin_fmaf(z[2 * j], MORE, -__uint_as_float(x & 0xFFFF0000u)),
                                                       (__bf16)__builtin_fmaf(z[2 * j + 1], MORE, -__uint_as_float(y & 0xFFFF0000u))});
          }
        }
        pf[m] = __builtin_bit_cast(Frag<VT>, uint4{w[0], w[1], w[2], w[3]});
        rest[m] = __builtin_bit_cast(Frag<VT>, uint4{d[0], d[1], d[2], d[3]});
      }
      if (masked) {  // (0 times what does not exist, or a new token that is not seen, may be NaN; what is seen is added at the end)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t k = (j / 4) * 16 + lg * 4 + j % 4;
#pragma unroll
          for (int b = 0; b < VB; ++b) {
            if (!(real >> k & 1)) vr[b][j] = Raw8<C>{};
            bad |= tame<C>(vr[b][j], t + k >= ctx);
          }
        }
      }
#pragma unroll
      for (int b = 0; b < VB; ++b) {
        auto step = [&]<int E>(std::integral_constant<int, E>) {
          const Frag<VT> vf = turned<C, VT, E>(vr[b]);
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            acc[m][b][E] = mma<VT>(vf, pf[m], acc[m][b][E]);
            acc[m][b][E] = mma<VT>(vf, rest[m], acc[m][b][E]);
          }
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

  if (C != GSK_I8) {
    const bool any = ballot64(bad != 0) != 0;
    if (lane == 0) sh.bad[wave] = any;
  }
  // What a row sees of the NaNs and infinities that were taken out, of the new tokens in this part, one by one: back from its own
  // token, which may lie in a later part.
  auto add_bad = [&](uint32_t h, uint32_t row, uint32_t e, float(&y)[8]) {
    const uint32_t i = row / p.group, low = max(k0, ctx);
    if (k1 <= low) return;
    for (uint32_t past = (a.parent ? ctx + i : min(ctx + i, k1 - 1)) + 1; past > low;) {
      const uint32_t t = past - 1;
      past = t;
      if (a.parent) {
        const int32_t node = sp.begin + (int32_t)(t - ctx), up = a.parent[node];
        past = up >= sp.begin && up < node ? ctx + (uint32_t)(up - sp.begin) + 1 : 0;
      }
      if (t >= k1) continue;
      const uint32_t pg = (uint32_t)a.table[(int64_t)r * a.table_ld + t / c.page];
      if (pg >= c.pages) continue;
      const int64_t at = (int64_t)pg * c.page_stride + (int64_t)(t % c.page) * c.token_stride + (int64_t)h * c.head_stride + e;
      float x[8];
      to_f32(load_raw8<C>((const char *)c.values + at * SZ), x);
#pragma unroll
      for (int d = 0; d < 8; ++d) y[d] += fabsf(x[d]) < INF ? 0.0f : x[d];
    }
  };

  // ---- the waves' results joined ------------------------------------------------------------------------------------------
  // A thread has eight elements of one of 16 rows. A part's scratch: rows x dim of O, then rows x (m, l).
  float *work = (float *)a.work;
  const int64_t part_size = (int64_t)p.rows * (c.dim + 2);
  // A share has two of them: of the request that it goes on with, and of the one that goes on after it.
  auto scratch = [&](uint32_t it, uint32_t h) {
    return work + (((int64_t)it * 2 + (it == first_item)) * c.heads + h) * part_size;
  };
  const uint32_t tr = tid / 16, te = tid % 16 * 8;
  auto finish = [&](uint32_t h, uint32_t row, uint32_t e, const float (&x)[8], float sum) {
    const uint32_t i = row / p.group, gi = row - i * p.group;
    const float inv = sum > 0 ? 1.0f / sum : 0.0f;
    float y[8];
#pragma unroll
    for (int d = 0; d < 8; ++d) y[d] = sum == 0 ? 0.0f : sum > 0 ? x[d] * inv : x[d] / sum;
    store_raw8<Q>((char *)a.out + (((int64_t)(sp.begin + i) * a.heads + h * p.group + gi) * c.dim + e) * 2, from_f32<Q>(y));
  };
#pragma unroll 1
  for (int m = 0; m < MT; ++m) {
    if (row0 + m * 16 >= rows) break;
#pragma unroll 1
    for (int b = 0; b < VB; ++b) {
      __syncthreads();  // (the last use of what lies there)
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
          const float sum = over_groups(l[mm], [](float x, float y) { return x + y; }) * MORE;
          if (lg == 0) {
            sh.m[wave][lc] = mx[mm];
            sh.l[wave][lc] = sum;
          }
        }
      }
      __syncthreads();
      const uint32_t row = row0 + m * 16 + tr, e = b * 128 + te;
      if (row >= rows || e >= c.dim) continue;
#pragma unroll 1
      for (uint32_t hh = 0; hh < heads_here; ++hh) {  // (four heads: a wave has all of one)
        float top = -INF, sum = 0, x[8] = {};
        const uint32_t w0 = four ? hh : 0, w1 = four ? hh + 1 : AW;
        for (uint32_t w = w0; w < w1; ++w) top = fmaxf(top, sh.m[w][tr]);
        for (uint32_t w = w0; w < w1; ++w) {
          if (sh.l[w][tr] == 0.0f) continue;
          const float f = weight_of(sh.m[w][tr], sh.l[w][tr], top);
          sum += f * sh.l[w][tr];
#pragma unroll
          for (int d = 0; d < 8; ++d) x[d] += f * sh.o[w][tr][te + d];
        }
        if (C != GSK_I8 && (sh.bad[0] | sh.bad[1] | sh.bad[2] | sh.bad[3])) add_bad(head0 + hh, row, e, x);
        if (parts == 1) {
          finish(head0 + hh, row, e, x, sum);
          continue;
        }
        float *o = scratch(item, head0 + hh) + (int64_t)(row - row0) * c.dim + e;
#pragma unroll
        for (int d = 0; d < 8; d += 2)
          st_ag((uint64_t *)(o + d), (uint64_t)__float_as_uint(x[d]) | (uint64_t)__float_as_uint(x[d + 1]) << 32);
        if (e == 0)
          st_ag((uint64_t *)(scratch(item, head0 + hh) + (int64_t)p.rows * c.dim + 2 * (row - row0)),
                (uint64_t)__float_as_uint(top) | (uint64_t)__float_as_uint(sum) << 32);
      }
    }
  }
  if (parts == 1) {
    __syncthreads();
    continue;
  }

  // ---- the parts joined ---------------------------------------------------------------------------------------------------
  store_wait();
  __syncthreads();
  uint32_t *tick = p.tick + (int64_t)first_item * each + x;  // (one turn at most goes on after a share)
  if (tid == 0) sh.last = ticket_add(tick) == parts - 1;
  __syncthreads();
  const bool last = sh.last;
  __syncthreads();
  if (!last) continue;
  if (tid == 0) st_ag(tick, 0u);
  // 16 threads a row again; with few rows, several such groups share a row's parts. A thread takes eight of its parts' loads at
  // once: a round trip, in most calls the only one.
#pragma unroll 1
  for (uint32_t mh = 0; mh < MT * heads_here; ++mh) {
    const uint32_t m = four ? 0 : mh, h = head0 + (four ? mh : 0);
    if (row0 + m * 16 >= rows) break;
    const uint32_t count = min(rows - row0 - m * 16, 16u), wide = count <= 1 ? 1 : 1u << (32 - __builtin_clz(count - 1));
    const uint32_t i = m * 16 + tr % wide, mine = tr / wide, shares = 16 / wide;
    const bool real = tr % wide < count;
#pragma unroll 1
    for (int b = 0; b < VB; ++b) {
      const uint32_t e = b * 128 + te;
      const bool in = real && e < c.dim;
      float top = -INF, sum = 0, y[8] = {};
      for (uint32_t s0 = mine; in && s0 < parts; s0 += 8 * shares) {
        uint64_t ml[8], w[8][4];
#pragma unroll
        for (uint32_t k = 0; k < 8; ++k) {
          const float *o = scratch(first_item + min(s0 + k * shares, parts - 1), h);
          ml[k] = ld_ag((const uint64_t *)(o + (int64_t)p.rows * c.dim + 2 * i));
#pragma unroll
          for (int d = 0; d < 4; ++d) w[k][d] = ld_ag((const uint64_t *)(o + (int64_t)i * c.dim + e) + d);
        }
        float next = top;
#pragma unroll
        for (uint32_t k = 0; k < 8; ++k) next = fmaxf(next, __uint_as_float((uint32_t)ml[k]));
        const float f = weight_of(top, sum, next);
        top = next;
        sum *= f;
#pragma unroll
        for (int d = 0; d < 8; ++d) y[d] *= f;
#pragma unroll
        for (uint32_t k = 0; k < 8; ++k) {
          const float part_l = __uint_as_float((uint32_t)(ml[k] >> 32));
          if (part_l == 0.0f || s0 + k * shares >= parts) continue;  // (nothing of this row in the part, or no such part)
          const float g = weight_of(__uint_as_float((uint32_t)ml[k]), part_l, top);
          sum += g * part_l;
#pragma unroll
          for (int d = 0; d < 4; ++d) {
            y[2 * d] += g * __uint_as_float((uint32_t)w[k][d]);
            y[2 * d + 1] += g * __uint_as_float((uint32_t)(w[k][d] >> 32));
          }
        }
      }
      if (shares > 1) {
        __syncthreads();
        *(f32x4 *)&sh.o[0][tr][te] = f32x4{y[0], y[1], y[2], y[3]};
        *(f32x4 *)&sh.o[0][tr][te + 4] = f32x4{y[4], y[5], y[6], y[7]};
        if (te == 0) {
          sh.m[0][tr] = top;
          sh.l[0][tr] = sum;
        }
        __syncthreads();
        if (in && mine == 0) {
          const float was = top;
          for (uint32_t k = 1; k < shares; ++k) top = fmaxf(top, sh.m[0][tr + k * wide]);
          const float f = weight_of(was, sum, top);
          sum *= f;
#pragma unroll
          for (int d = 0; d < 8; ++d) y[d] *= f;
          for (uint32_t k = 1; k < shares; ++k) {
            const float part_l = sh.l[0][tr + k * wide], g = weight_of(sh.m[0][tr + k * wide], part_l, top);
            if (part_l == 0.0f) continue;
            sum += g * part_l;
#pragma unroll
            for (int d = 0; d < 8; ++d) y[d] += g * sh.o[0][tr + k * wide][te + d];
          }
        }
      }
      if (in && mine == 0) finish(h, row0 + i, e, y, sum);
    }
  }
  __syncthreads();
  }
}

template <uint32_t Q, uint32_t C>
void launch_attend_types(const AttendArgs &p, int mt, dim3 grid, hipStream_t s) {
  auto go = [&](auto kd, auto m) { hipLaunchKernelGGL((attend_kernel<Q, C, kd(), m()>), grid, dim3(AT), 0, s, p); };
  auto by = [&](auto kd) {
    if (mt == 1) go(kd, std::integral_constant<int, 1>{});
    else if (mt == 2) go(kd, std::integral_constant<int, 2>{});
    else if constexpr (kd() <= 4) go(kd, std::integral_constant<int, 3>{});
  };
  if (p.c.dim <= 64) by(std::integral_constant<int, 2>{});
  else if (p.c.dim <= 96) by(std::integral_constant<int, 3>{});
  else if (p.c.dim <= 128) by(std::integral_constant<int, 4>{});
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
