// Products of rows sorted by expert: which kernel.
#include "kernels.h"

using namespace lutmoe;

namespace lutmoe_host {

int launch_grouped(const GroupedArgs& g, hipStream_t s) {
    if (g.op == kGroupedFwd && grouped_few_rows(g)) return launch_grouped_few(g, s);
    if (g.op == kGroupedFwd && g.w_scales && !g.x_scales) return launch_grouped_mx(g, s);
    return launch_grouped_tile(g, s);
}

}  // namespace lutmoe_host
