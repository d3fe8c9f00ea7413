// Layer norm of bfloat16 rows.
#include "nb_layer_norm_launch.cuh"

namespace nbtrain {

template int ln_forward<__nv_bfloat16>(const LnForward& a);
template int ln_backward<__nv_bfloat16>(const LnBackward& a);

}  // namespace nbtrain
