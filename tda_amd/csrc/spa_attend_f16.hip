// spa_attend_f16.hip -- spa_attend.hpp for float16.
#include "spa_attend.hpp"

namespace spa {

int launch_attend_f16(const AttendParams& p, int d, int dv, void* stream) { return pick<sda::TrH>(p, d, dv, stream); }

}  // namespace spa
