// The group norm kernels of one element type (group_norm.h).
#include <type_traits>

#define M355_GN_T float
#define M355_GN_RUN run_f32
#include "group_norm_types.h"
