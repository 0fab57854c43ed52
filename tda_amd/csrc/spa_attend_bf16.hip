// spa_attend_bf16.hip -- spa_attend.hpp for bfloat16.
#include "spa_attend.hpp"

namespace spa {

int launch_attend_bf16(const AttendParams& p, int d, int dv, void* stream) { return pick<sda::TrB>(p, d, dv, stream); }

}  // namespace spa
