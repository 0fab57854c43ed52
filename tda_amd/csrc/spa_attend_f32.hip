// spa_attend_f32.hip -- spa_attend.hpp for float32 (a file a type, so that they compile side by side).
#include "spa_attend.hpp"

namespace spa {

int launch_attend_f32(const AttendParams& p, int d, int dv, void* stream) { return pick<sda::TrF>(p, d, dv, stream); }
int launch_attend(const AttendParams& p, int dtype, int d, int dv, void* stream) {
  return dtype == 0 ? launch_attend_f32(p, d, dv, stream) : dtype == 1 ? launch_attend_bf16(p, d, dv, stream) : launch_attend_f16(p, d, dv, stream);
}

}  // namespace spa
