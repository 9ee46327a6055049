// The plan and the launches of gsk_attend (include/gsk.h); the kernel is in gsk_attend_body.h.
#include "gsk_attend_body.h"

namespace gse {

namespace {

// MT of the kernel: as many of a request's rows as share a tile's loads, up to 48. 96 trees of 36 rows a head: 250 us with 3, 283 with
// tiles of 2 (which read the cache twice), 338 of 1; of 18 rows: 228 with 2, 239 with 3, 291 with 1; 24 chains of up to 18: 27.2 with 2,
// 29.3 with 1, 32.5 with 3.
int row_tiles(const gsk_cache &c, const gsk_attention &a) {
  const uint64_t rows = (uint64_t)a.max_new * (a.heads / c.heads);
  return rows <= 16 ? 1 : rows <= 32 || c.dim > 128 ? 2 : 3;
}

}  // namespace

uint64_t attend_tiles(const gsk_cache &c, const gsk_attention &a) {
  const uint64_t rows = (uint64_t)std::min(a.max_new, a.tokens) * (a.heads / c.heads), most = 16 * row_tiles(c, a);
  return std::max((rows + most - 1) / most, (uint64_t)1);
}

AttendPlan attend_plan(const gsk_cache &c, const gsk_attention &a, uint32_t tickets, int cus) {
  const uint64_t rows = (uint64_t)a.max_new * (a.heads / c.heads), most = 16 * row_tiles(c, a);
  AttendPlan p;
  const uint64_t tiles = attend_tiles(c, a);
  // One round of workgroups, as many on each XCD, if the requests' longest tables fill it.
  const uint64_t xcd = (uint64_t)cus / 8 * attend_resident(c.dim <= 128 ? 4 : 8, row_tiles(c, a));
  const uint64_t blocks = a.requests * tiles * (TURN + ((uint64_t)a.max_pages * c.page + AB - 1) / AB);
  auto round = [&](uint64_t each) { return std::min(each <= xcd ? xcd / each * 8 : xcd * 8 / each, (uint64_t)tickets / each); };
  p.items = (uint32_t)std::max(std::min(round(c.heads), blocks / SHARE_MIN), (uint64_t)1);
  // Four heads a workgroup, where heads of at most 128 bytes lie next to each other in a token: its loads are then four times as
  // long a piece of memory (8-bit rows of 128 bytes, 128 requests of up to 16384 tokens: 637 -> 553 us, 534 since waves give way; 64:
  // 337 -> 310; with the heads ahead 481 as it is; rows of 256 bytes: 529 -> 538). The parts of a request are then four times as
  // many, joined by a quarter of the workgroups: not where a request has more than about six (32 such requests: 180 us, 212 so; 8 of
  // 131072: 299, 428).
  const bool together = c.heads % AW == 0 && most == 16 && c.head_stride < c.token_stride && c.dim * (c.type >= GSK_E4M3 ? 1 : 2) <= 128;
  p.items4 = together ? (uint32_t)round((uint64_t)c.heads / AW) : 0;
  if (p.items4 > 6 * (uint64_t)a.requests) p.items4 = 0;
  if (blocks < (uint64_t)p.items4 * FOUR_MIN) p.items4 = 0;
  const uint64_t shares = std::max(p.items, p.items4);
  p.work = shares == 1 ? 0 : (int64_t)(shares * 2 * c.heads * std::min(rows, most) * (c.dim + 2) * sizeof(float));
  return p;
}

hipError_t launch_attend(const gsk_cache &c, const gsk_attention &a, const AttendPlan &plan, uint32_t *tick, hipStream_t s) {
  AttendArgs p;
  p.c = c;
  p.a = a;
  p.items = plan.items;
  p.items4 = plan.items4;
  p.group = a.heads / c.heads;
  const int mt = row_tiles(c, a);
  p.rows = (uint32_t)std::min((uint64_t)a.max_new * p.group, (uint64_t)(16 * mt));
  p.tick = tick;
  const uint64_t blocks = std::max(((uint64_t)p.items + 7) / 8 * 8 * c.heads, ((uint64_t)p.items4 + 7) / 8 * 8 * (c.heads / AW));
  if (blocks > INT32_MAX) return hipErrorInvalidValue;
  const dim3 grid((uint32_t)blocks);
  const bool half = a.type == GSK_F16;
  if (c.type == GSK_E4M3) (half ? launch_attend_f16_e4m3 : launch_attend_bf16_e4m3)(p, mt, grid, s);
  else if (c.type == GSK_I8) (half ? launch_attend_f16_i8 : launch_attend_bf16_i8)(p, mt, grid, s);
  else (half ? launch_attend_f16 : launch_attend_bf16)(p, mt, grid, s);
  return hipGetLastError();
}

}  // namespace gse
