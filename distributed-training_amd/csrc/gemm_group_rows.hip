// Group and statistics kernels of few rows.
#include "gemm_group_tiles.h"

namespace dtmi {

template void launch_group_rows<float>(const GroupArgs&, int, int, int);
template void launch_group_rows<double>(const GroupArgs&, int, int, int);
template void launch_stats_rows<float>(const StatsArgs&, int, int, int);
template void launch_stats_rows<double>(const StatsArgs&, int, int, int);

}  // namespace dtmi
