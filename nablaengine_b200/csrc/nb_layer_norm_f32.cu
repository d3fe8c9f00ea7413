// Layer norm of float32 rows.
#include "nb_layer_norm_launch.cuh"

namespace nbtrain {

long long ln_max_parts(long long rows, int cols) {
  const int wide = ln_wide_parts(rows);
  if (cols > LN_MAX_COLS) return wide;
  int lanes, ept;
  ln_spread(cols, true, &lanes, &ept);
  const long long blocks = (rows * lanes + 255) / 256;  // (blocks of 256 threads or more, two per SM at most)
  return std::max<long long>(std::min<long long>(blocks, 2 * SMS), wide);
}

template int ln_forward<float>(const LnForward& a);
template int ln_backward<float>(const LnBackward& a);

}  // namespace nbtrain
