// Launch wrappers of the operators of include/gsk.h.
#pragma once
#include "../../include/gsk.h"
#include "gse_int.h"

namespace gse {

hipError_t launch_write(const gsk_cache &c, const gsk_rows &a, hipStream_t s);
hipError_t launch_read(const gsk_cache &c, const gsk_read_rows &a, hipStream_t s);
hipError_t launch_reorder(const gsk_reorder_beams &a, hipStream_t s);

// How a call of gsk_attend is cut (gsk_attend.hip); tick: the tickets that it may use.
struct AttendPlan {
  uint32_t items;  // equal shares of the work on the requests' cached tokens: workgroups per cache head, at most
  uint32_t items4; // shares where a workgroup takes four heads (0: it never does)
  int64_t work;    // scratch bytes
};
uint64_t attend_tiles(const gsk_cache &c, const gsk_attention &a);  // of a request's (new token, query head of the group) rows
AttendPlan attend_plan(const gsk_cache &c, const gsk_attention &a, uint32_t tickets, int cus);
hipError_t launch_attend(const gsk_cache &c, const gsk_attention &a, const AttendPlan &p, uint32_t *tick, hipStream_t s);

int64_t beam_work(const gsk_beams &a, int cus);
hipError_t launch_beam(const gsk_beams &a, int cus, uint32_t *tick, uint32_t tickets, hipStream_t s);

}  // namespace gse
