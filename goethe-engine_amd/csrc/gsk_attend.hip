// Attention of a step's new tokens over the paged cache (gsk_attend, include/gsk.h).
#include "gsk_dev.h"
#include "gsk_int.h"

namespace gse {

namespace {

constexpr int AT = 256;

// A workgroup a (request, new token, query head): 16 groups of 16 lanes take the cached tokens in turn, a lane eight (sixteen)
// elements of each, with a running maximum and sum per group; joined in LDS at the end.
template <uint32_t Q, uint32_t C>
__global__ __launch_bounds__(AT) void attend_kernel(gsk_cache c, gsk_attention a, uint32_t r0) {
  __shared__ float o[16][GSK_MAX_DIM], ms[16], ls[16];
  const uint32_t r = r0 + blockIdx.z, i = blockIdx.y, hq = blockIdx.x, tid = threadIdx.x, grp = tid / 16, j = tid % 16;
  const int64_t b = a.begin ? a.begin[r] : r, e = a.begin ? a.begin[r + 1] : b + 1, len = a.seq_len[r], n = e - b;
  if (b < 0 || e > (int64_t)a.tokens || (int64_t)i >= n) return;
  const int64_t row = b + i, ctx = len - n;
  const bool ok = !(a.status && a.status[r]) && ctx >= 0 && len <= (int64_t)a.max_pages * c.page;
  uint64_t path = 0;
  if (a.parent) {
    for (int64_t at = row;;) {
      path |= 1ull << (at - b);
      const int64_t up = a.parent[at];
      if (up < b || up >= at) break;
      at = up;
    }
  }
  const uint32_t h = hq / (a.heads / c.heads);
  float q[2][8] = {}, acc[2][8] = {}, m = -INFINITY, l = 0;
  const char *qp = (const char *)a.q + (row * a.q_token_stride + hq * a.q_head_stride) * 2;
  for (int k = 0; k < 2; ++k)
    if (k * 128 + j * 8 < c.dim) to_f32(load_raw8<Q>(qp + (k * 128 + j * 8) * 2), q[k]);
  const int64_t end = ok ? (a.parent ? len : ctx + i + 1) : 0;
  for (int64_t t = grp; t < end; t += 16) {
    if (t >= ctx && a.parent && !(path >> (t - ctx) & 1)) continue;
    const uint32_t pi = (uint32_t)t / c.page, pg = (uint32_t)a.table[r * a.table_ld + pi];
    if (pg >= c.pages) continue;
    const uint32_t off = (uint32_t)t - pi * c.page;
    const int64_t at = (int64_t)pg * c.page_stride + off * c.token_stride + h * c.head_stride;
    const int64_t st = (int64_t)pg * c.scale_page_stride + off * c.scale_token_stride + h * c.scale_head_stride;
    float s = 0, v[2][8] = {};
    for (int k = 0; k < 2; ++k) {
      if (k * 128 + j * 8 < c.dim) {
        float x[8];
        to_f32(load_raw8<C>((const char *)c.keys + (at + k * 128 + j * 8) * type_size<C>), x);
        for (int d = 0; d < 8; ++d) s += q[k][d] * x[d];
        to_f32(load_raw8<C>((const char *)c.values + (at + k * 128 + j * 8) * type_size<C>), v[k]);
      }
    }
    for (int k = 8; k > 0; k /= 2) s += __shfl_xor(s, k, WAVE);
    s *= a.scale;
    float vs = 1;
    if constexpr (type_is_8bit<C>) {
      s *= c.key_scales[st];
      vs = c.value_scales[st];
    }
    if (s == -INFINITY) continue;
    const float m2 = fmaxf(m, s), f = __expf(m - m2), p = __expf(s - m2);
    m = m2;
    l = l * f + p;
    for (int k = 0; k < 2; ++k)
      for (int d = 0; d < 8; ++d) acc[k][d] = acc[k][d] * f + p * vs * v[k][d];
  }
  for (int k = 0; k < 2; ++k)
    for (int d = 0; d < 8; ++d) o[grp][k * 128 + j * 8 + d] = acc[k][d];
  ms[grp] = m;
  ls[grp] = l;
  __syncthreads();
  if (tid >= c.dim) return;
  float top = -INFINITY, sum = 0, x = 0;
  for (int k = 0; k < 16; ++k) top = fmaxf(top, ms[k]);
  for (int k = 0; k < 16; ++k) {
    if (ls[k] == 0) continue;
    const float f = __expf(ms[k] - top);
    sum += f * ls[k];
    x += f * o[k][tid];
  }
  x = sum == 0 ? 0 : x / sum;
  const int64_t at = (row * a.heads + hq) * c.dim + tid;
  if constexpr (Q == GSK_BF16) ((__bf16 *)a.out)[at] = (__bf16)x;
  else ((_Float16 *)a.out)[at] = (_Float16)x;
}

}  // namespace

AttendPlan attend_plan(const gsk_cache &, const gsk_attention &, uint32_t, int) { return {1, 1, 0}; }

hipError_t launch_attend(const gsk_cache &c, const gsk_attention &a, const AttendPlan &, uint32_t *, hipStream_t s) {
  auto go = [&](auto q, auto k) {
    for (uint32_t r0 = 0; r0 < a.requests; r0 += 65535)
      hipLaunchKernelGGL((attend_kernel<q(), k()>), dim3(a.heads, a.max_new, min(a.requests - r0, 65535u)), dim3(AT), 0, s, c, a, r0);
  };
  auto by = [&](auto q) {
    if (c.type == GSK_E4M3) go(q, std::integral_constant<uint32_t, GSK_E4M3>{});
    else if (c.type == GSK_I8) go(q, std::integral_constant<uint32_t, GSK_I8>{});
    else go(q, q);
  };
  if (a.type == GSK_BF16) by(std::integral_constant<uint32_t, GSK_BF16>{});
  else by(std::integral_constant<uint32_t, GSK_F16>{});
  return hipGetLastError();
}

}  // namespace gse
