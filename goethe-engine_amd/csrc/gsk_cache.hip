// The paged cache's rows (include/gsk.h): written (gsk_write), read back (gsk_read), moved between beams (gsk_reorder).
#include "gsk_dev.h"
#include "gsk_int.h"

namespace gse {

namespace {

// ---- write ---------------------------------------------------------------------------------------------------------------
// A group of 8, 16 or 32 lanes owns one token's head of the keys or of the values, a lane eight elements of it; in 8 bits the
// group finds the row's largest magnitude by exchanges within it. Rows with a NaN or an infinity are found with it: as unsigned
// integers their magnitudes are the largest.
//
// Bound: up to some hundreds of tokens the launch and two dependent reads (64 tokens of 8 heads of 128: 2.4 us); from there memory:
// 16384 tokens of 5 heads of 80, fp16 into 8-bit integers (39 MB), 12.5 us or 3.1 TB/s, 65536 of them 38.5 us or 4.1 TB/s. A group
// with four rows in turn, all loaded first, took as long at both.
constexpr int CT = 256;

struct Place {
  int64_t at, scale;  // element offsets of the row and of its scale
};
__device__ __forceinline__ Place place(const gsk_cache &c, uint32_t pg, uint32_t off, uint32_t head) {
  return {(int64_t)pg * c.page_stride + (int64_t)off * c.token_stride + (int64_t)head * c.head_stride,
          (int64_t)pg * c.scale_page_stride + (int64_t)off * c.scale_token_stride + (int64_t)head * c.scale_head_stride};
}

template <uint32_t SRC, uint32_t DST, int GL>
__global__ __launch_bounds__(CT) void write_kernel(gsk_cache c, gsk_rows a, Div heads, Div page) {
  const uint32_t j = threadIdx.x % GL, id = blockIdx.x * (CT / GL) + threadIdx.x / GL;
  if (id >= a.tokens * c.heads) return;  // (the group as a whole)
  const bool values = blockIdx.y != 0, mine = j * 8 < c.dim;
  const char *src = (const char *)(values ? a.v : a.k) + j * 8 * type_size<SRC>;
  const int64_t ts = values ? a.v_token_stride : a.k_token_stride, hs = values ? a.v_head_stride : a.k_head_stride;
  char *dst = (char *)(values ? c.values : c.keys) + j * 8 * type_size<DST>;
  float *scales = values ? c.value_scales : c.key_scales;
  uint32_t head, off;
  const uint32_t t = quotient(id, heads, head);
  const uint64_t slot = (uint64_t)a.slot[t];
  Raw8<SRC> raw{};
  if (mine) raw = load_raw8<SRC>(src + ((int64_t)t * ts + (int64_t)head * hs) * type_size<SRC>);
  if (slot >= (uint64_t)c.pages * c.page) return;  // (negative ones are past it; the group as a whole)
  const uint32_t pg = quotient((uint32_t)slot, page, off);
  const Place p = place(c, pg, off, head);
  float x[8];
  to_f32(raw, x);
  if constexpr (type_is_8bit<DST>) {
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) m = max(m, __float_as_uint(x[e]) & 0x7FFFFFFFu);
    m = group_max<GL>(m);
    const bool bad = m >= 0x7F800000u;
    const float most = DST == GSK_E4M3 ? 1.0f / 448.0f : 1.0f / 127.0f;
    const float scale = fmaxf(__fmul_rn(__uint_as_float(m), most), 0x1p-126f), inv = __fdiv_rn(1.0f, scale);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = bad ? 0.0f : __fmul_rn(x[e], inv);
    if (j == 0) scales[p.scale] = bad ? __uint_as_float(0x7FC00000u) : scale;
  }
  if (mine) store_raw8<DST>(dst + p.at * type_size<DST>, from_f32<DST>(x));
}

// ---- read ----------------------------------------------------------------------------------------------------------------
// A workgroup takes `tokens` rows, every head of them, keys and values. Its first wave finds their places (a lane a token: the
// request by a search of the whole wave for the first, from there on step by step; then the page) and leaves them in LDS; the
// threads then walk the rows' pieces of eight elements, which lie together in the output.
//
// Bound: memory. 32 requests of 4096 to 8192 tokens of 5 heads of 80, 8-bit integers to fp16 (168 MB read, 281 written by the
// counters): 94 us, 4.4 TB/s. 4 requests of 256 to 512 tokens: 4.3 us, the search, the table and the rows one after the other.
constexpr uint32_t RTOK = 32;  // tokens of a workgroup, at most

struct ReadShared {
  int64_t at[RTOK], scale[RTOK];
  int32_t kind[RTOK];  // 1: a cached token, 0: zeros, -1: left as it is
};

template <uint32_t SRC, uint32_t DST, int U>
__global__ __launch_bounds__(CT) void read_kernel(gsk_cache c, gsk_read_rows a, uint32_t tokens, Div by_pieces, Div by_heads) {
  __shared__ ReadShared sh;
  const uint32_t tid = threadIdx.x, row0 = blockIdx.x * tokens, pieces = c.dim / 8;
  if (tid < WAVE) {
    uint32_t r = wave_find(a.begin, a.requests, row0);
    const uint32_t row = row0 + tid;
    if (tid < tokens) {
      int32_t kind = -1;
      Place p = {0, 0};
      if (row < a.rows) {
        int64_t b = a.begin[r], e = a.begin[r + 1];
        while (e <= (int64_t)row && r + 1 < a.requests) {
          ++r;
          b = e;
          e = a.begin[r + 1];
        }
        if ((int64_t)row >= b && (int64_t)row < e) {
          const int64_t t = (a.first ? a.first[r] : 0) + ((int64_t)row - b);
          kind = 0;
          if (t >= 0 && t < (int64_t)a.max_pages * c.page) {
            const uint32_t pi = (uint32_t)t / c.page, pg = (uint32_t)a.table[(int64_t)r * a.table_ld + pi];
            if (pg < c.pages) {
              kind = 1;
              p = place(c, pg, (uint32_t)t - pi * c.page, 0);
            }
          }
        }
      }
      sh.kind[tid] = kind;
      sh.at[tid] = p.at;
      sh.scale[tid] = p.scale;
    }
  }
  __syncthreads();
  const uint32_t n = min(tokens, a.rows - row0) * c.heads * pieces;
  const int64_t out = (int64_t)row0 * c.heads * pieces;
  for (uint32_t i0 = tid; i0 < n; i0 += U * CT) {
    Raw8<SRC> raw[U][2];
    float scale[U][2];
    int32_t kind[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t i = min(i0 + u * CT, n - 1);
      uint32_t piece, head;
      const uint32_t t = quotient(quotient(i, by_pieces, piece), by_heads, head);
      kind[u] = i0 + u * CT < n ? sh.kind[t] : -1;  // (a token without a place reads slot 0)
      const int64_t at = sh.at[t] + (int64_t)head * c.head_stride + piece * 8;
      raw[u][0] = load_raw8<SRC>((const char *)c.keys + at * type_size<SRC>);
      raw[u][1] = load_raw8<SRC>((const char *)c.values + at * type_size<SRC>);
      if constexpr (type_is_8bit<SRC>) {
        const int64_t sc = sh.scale[t] + (int64_t)head * c.scale_head_stride;
        scale[u][0] = c.key_scales[sc];
        scale[u][1] = c.value_scales[sc];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (kind[u] < 0) continue;
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        float x[8];
        to_f32(raw[u][v], x);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if constexpr (type_is_8bit<SRC>) x[e] = __fmul_rn(x[e], scale[u][v]);
          x[e] = kind[u] ? x[e] : 0.0f;
        }
        store_raw8<DST>((char *)(v ? a.v : a.k) + (out + i0 + u * CT) * 8 * type_size<DST>, from_f32<DST>(x));
      }
    }
  }
}

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// ---- reorder --------------------------------------------------------------------------------------------------------------
// A thread owns one vector of one token of one cache, in every beam of a group: it loads the vectors of all beams that move
// before it stores any, so that the beams are permuted in place without a copy; no vector belongs to two threads. A workgroup
// finds the offsets of TB tokens (a thread a token's beam) and leaves them in LDS, the moving beams of a token one after the
// other; then its threads walk the (cache, chunk, token, place) of the block: neighbouring tokens of a chunk lie together
// where the heads come first.
//
// Bound: memory where there is enough to move (8 groups of 8 beams, 256 tokens in 48 caches of 400 bytes: 550 MB, 121 to 125 us over two
// or three sets of arrays in turn, 4.5 TB/s; 99 us where calls repeat on one set, part of which the last-level cache holds); else the
// launch, the table and the rows one after the other (4 beams, 16 tokens, 64 caches of 2 KB rows: 6.5 us in turn, 6.0 on one set).
struct ReorderShared {
  int64_t src[CT], dst[CT];
  uint32_t n[CT];
};

template <typename VEC, int MB>
__global__ __launch_bounds__(CT) void reorder_kernel(gsk_reorder_beams a, Div vecs, Div chunks) {
  __shared__ ReorderShared sh;
  constexpr uint32_t TB = CT / MB;  // tokens of a block
  const uint32_t g = blockIdx.z, tid = threadIdx.x, beam = tid % MB, tok = tid / MB;
  const uint32_t row = g * a.beams + beam;
  const int64_t first = a.first ? a.first[g] : 0;
  int64_t len = 0;
  uint32_t from = row;
  if (beam < a.beams) {
    const uint32_t p = (uint32_t)a.parent[row];
    if (p < a.beams) from = g * a.beams + p;
    len = min(a.seq_len[row], a.seq_len[from]);
  }
  const bool moves = from != row && first >= 0;
  const int64_t most = min((int64_t)wave_max_u64(moves && len > 0 ? (uint64_t)len : 0), (int64_t)a.max_pages * a.page);
  const uint32_t columns = a.caches * a.chunks * TB * vecs.d;
  for (int64_t t0 = first + (int64_t)blockIdx.y * TB; t0 < most; t0 += (int64_t)gridDim.y * TB) {
    const int64_t t = t0 + tok;
    uint32_t ps = 0, pd = 0, off = 0;
    bool go = moves && t < len && t < most;
    if (go) {
      const uint32_t pi = (uint32_t)t / a.page;
      off = (uint32_t)t - pi * a.page;
      ps = (uint32_t)a.table[(int64_t)from * a.table_ld + pi];
      pd = (uint32_t)a.table[(int64_t)row * a.table_ld + pi];
      go = ps < a.pages && pd < a.pages;
    }
    const uint64_t all = ballot64(go), mine = MB == 64 ? all : (all >> (lane_id() / MB * MB)) & ((1ull << MB) - 1);
    __syncthreads();  // (the block before is done)
    if (go) {
      const uint32_t k = tok * MB + (uint32_t)__popcll(mine & ((1ull << beam) - 1));
      sh.src[k] = (int64_t)ps * a.page_stride + (int64_t)off * a.token_stride;
      sh.dst[k] = (int64_t)pd * a.page_stride + (int64_t)off * a.token_stride;
    }
    if (beam == 0) sh.n[tok] = (uint32_t)__popcll(mine);
    __syncthreads();
    for (uint32_t id = blockIdx.x * CT + tid; id < columns; id += gridDim.x * CT) {
      uint32_t place, chunk;
      const uint32_t x = quotient(id, vecs, place), k = quotient(x / TB, chunks, chunk), to = x % TB, n = sh.n[to];
      if (n == 0) continue;
      char *base = a.cache_ptrs ? (char *)a.cache_ptrs[k] : (char *)a.cache + k * a.cache_stride;
      base += (int64_t)chunk * a.chunk_stride + (int64_t)place * sizeof(VEC);
      VEC v[MB];
#pragma unroll
      for (uint32_t e = 0; e < MB; ++e)
        if (e < n) v[e] = *(const VEC *)(base + sh.src[to * MB + e]);
#pragma unroll
      for (uint32_t e = 0; e < MB; ++e)
        if (e < n) *(VEC *)(base + sh.dst[to * MB + e]) = v[e];
    }
  }
}

template <typename F>
void by_lanes(uint32_t dim, F f) {
  if (dim <= 64) f(std::integral_constant<int, 8>{});
  else if (dim <= 128) f(std::integral_constant<int, 16>{});
  else f(std::integral_constant<int, 32>{});
}
template <typename F>
void by_type(uint32_t t, F f) {
  switch (t) {
    case GSK_BF16: return f(std::integral_constant<uint32_t, GSK_BF16>{});
    case GSK_F16: return f(std::integral_constant<uint32_t, GSK_F16>{});
    case GSK_F32: return f(std::integral_constant<uint32_t, GSK_F32>{});
    case GSK_E4M3: return f(std::integral_constant<uint32_t, GSK_E4M3>{});
    default: return f(std::integral_constant<uint32_t, GSK_I8>{});
  }
}

}  // namespace

hipError_t launch_write(const gsk_cache &c, const gsk_rows &a, hipStream_t s) {
  by_type(a.type, [&](auto src) {
    by_type(c.type, [&](auto dst) {
      if constexpr (!type_is_8bit<src()> && dst() != GSK_F32) {
        by_lanes(c.dim, [&](auto gl) {
          const uint64_t rows = (uint64_t)a.tokens * c.heads, each = CT / gl();
          hipLaunchKernelGGL((write_kernel<src(), dst(), gl()>), dim3((uint32_t)((rows + each - 1) / each), 2), dim3(CT), 0, s, c, a,
                             div_by(c.heads), div_by(c.page));
        });
      }
    });
  });
  return hipGetLastError();
}

hipError_t launch_read(const gsk_cache &c, const gsk_read_rows &a, hipStream_t s) {
  // tokens of a workgroup: as many as leave the launch 2048 of them (8 requests of up to 1024 tokens: 8.7 us, with 8192 workgroups
  // 10.1; up to 4096 tokens: 23.2, with 8192 workgroups 25.3, with 512 24.0)
  uint32_t tokens = 1;
  while (tokens < RTOK && a.rows / tokens >= 4096) tokens *= 2;
  const uint32_t pieces = c.dim / 8;
  by_type(c.type, [&](auto src) {
    by_type(a.type, [&](auto dst) {
      if constexpr (src() != GSK_F32 && !type_is_8bit<dst()>) {
        auto go = [&](auto u) {
          hipLaunchKernelGGL((read_kernel<src(), dst(), u()>), dim3((a.rows + tokens - 1) / tokens), dim3(CT), 0, s, c, a, tokens,
                             div_by(pieces), div_by(c.heads));
        };
        // four pieces a thread at once where its workgroup has them: 32 requests of up to 8192 tokens 97 us, one by one 101; with
        // fewer the lanes past the end cost (8 of up to 1024: 8.7 us, 10.4 so)
        if ((uint64_t)tokens * c.heads * pieces >= 4 * CT) go(std::integral_constant<int, 4>{});
        else go(std::integral_constant<int, 1>{});
      }
    });
  });
  return hipGetLastError();
}

hipError_t launch_reorder(const gsk_reorder_beams &in, hipStream_t s) {
  // Workgroups of a launch to aim for, a thread's vectors of a block of tokens (calls on one set of arrays; 8 x 8 beams, 256 and
  // 16 tokens: 98 and 8.9 us; with four vectors 107 and 13.2, with two 103 and 10.3; with 2048 workgroups 101 and 8.1, with 8192
  // 95 and 9.9, and 4 beams of 16 tokens 5.5, 5.8 and 7.2 with 2048, 4096 and 8192).
  constexpr int64_t WGS = 4096, EACH = 1;
  auto go = [&](auto v, auto mb) {
    using V = decltype(v);
    constexpr int MB = mb();
    const uint32_t vecs = (uint32_t)(in.chunk_bytes / sizeof(V));
    const int64_t columns = (int64_t)in.caches * in.chunks * (CT / MB) * vecs;  // (below 2^32)
    const int64_t blocks = ((int64_t)in.max_pages * in.page + CT / MB - 1) / (CT / MB);
    for (uint32_t g0 = 0; g0 < in.groups; g0 += 65535) {
      gsk_reorder_beams a = in;
      a.groups = std::min(in.groups - g0, 65535u);
      a.table += (int64_t)g0 * in.beams * in.table_ld;
      a.seq_len += (int64_t)g0 * in.beams;
      a.parent += (int64_t)g0 * in.beams;
      if (a.first) a.first += g0;
      const int64_t x = std::max(std::min((columns + EACH * CT - 1) / (EACH * CT), WGS / a.groups), (int64_t)1);
      const int64_t y = std::min(std::min(blocks, (int64_t)65535), std::max((int64_t)1, WGS / (a.groups * x)));
      hipLaunchKernelGGL((reorder_kernel<V, MB>), dim3((uint32_t)x, (uint32_t)y, a.groups), dim3(CT), 0, s, a, div_by(vecs),
                         div_by(in.chunks));
    }
  };
  auto by_beams = [&](auto v) {
    if (in.beams <= 4) go(v, std::integral_constant<int, 4>{});
    else if (in.beams <= 8) go(v, std::integral_constant<int, 8>{});
    else if (in.beams <= 16) go(v, std::integral_constant<int, 16>{});
    else go(v, std::integral_constant<int, 32>{});
  };
  // the widest vector that every address is a multiple of
  const uint64_t all = (uint64_t)in.chunk_bytes | (uint64_t)in.page_stride | (uint64_t)in.token_stride | (uint64_t)in.chunk_stride |
                       (in.cache_ptrs ? (uint64_t)in.align : (uint64_t)in.cache | (uint64_t)in.cache_stride);
  if (all % 16 == 0) by_beams(u32x4{});
  else if (all % 4 == 0) by_beams(uint32_t{});
  else by_beams(uint8_t{});
  return hipGetLastError();
}

}  // namespace gse
