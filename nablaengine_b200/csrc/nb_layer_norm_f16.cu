// Layer norm of float16 rows.
#include "nb_layer_norm_launch.cuh"

namespace nbtrain {

template int ln_forward<__half>(const LnForward& a);
template int ln_backward<__half>(const LnBackward& a);

}  // namespace nbtrain
