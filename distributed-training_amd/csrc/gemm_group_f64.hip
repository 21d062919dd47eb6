// float64 group and statistics kernels on 128 x 128 block tiles.
#include "gemm_group_tiles.h"

namespace dtmi {

template void launch_group<double, 128>(const GroupArgs&, int, int, bool);
template void launch_stats<double, 128>(const StatsArgs&, int, bool);

}  // namespace dtmi
