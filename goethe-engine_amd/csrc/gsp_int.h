// Launch wrappers of the operators of include/gsp.h.
#pragma once
#include "../../include/gsp.h"
#include "gse_int.h"

namespace gse {

bool chains_fit(const RowsWs &w, const gsp_chains &c);  // whether a row's segment sums fit the workspace
hipError_t launch_chains(const RowsWs &w, const gsp_chains &c, hipStream_t s);
hipError_t launch_pages(const gsp_pages &p, const gsp_step &t, hipStream_t s);
hipError_t launch_path(const gsp_path &p, hipStream_t s);

}  // namespace gse
