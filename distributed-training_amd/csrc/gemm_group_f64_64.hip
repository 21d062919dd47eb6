// float64 group and statistics kernels on 64 x 64 block tiles.
#include "gemm_group_tiles.h"

namespace dtmi {

template void launch_group<double, 64>(const GroupArgs&, int, int, bool);
template void launch_stats<double, 64>(const StatsArgs&, int, bool);

}  // namespace dtmi
