// Group and statistics kernels of small products, on 32 x 32 tiles.
#include "gemm_group_tiles.h"

namespace dtmi {

template void launch_group_direct<float>(const GroupArgs&, int, int, int);
template void launch_group_direct<double>(const GroupArgs&, int, int, int);
template void launch_stats_direct<float>(const StatsArgs&, int, int);
template void launch_stats_direct<double>(const StatsArgs&, int, int);

}  // namespace dtmi
