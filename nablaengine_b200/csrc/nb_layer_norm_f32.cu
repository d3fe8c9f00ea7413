// Layer norm of float32 rows.
#include "nb_layer_norm_launch.cuh"

namespace nbtrain {

long long ln_max_parts(long long rows, int cols) {
  const int wide = ln_wide_parts(rows);
  if (cols > LN_WIDEST) return wide;
  LnTiles t;  // (the teams of either value size: rows / groups, two blocks per SM at most)
  ln_spread(cols, 4, true, &t);
  const long long teams = (rows * t.lanes + 255) / 256;
  return std::max<long long>(std::min<long long>(teams, 2 * SMS), wide);
}

template int ln_forward<float>(const LnForward& a);
template int ln_backward<float>(const LnBackward& a);

}  // namespace nbtrain
