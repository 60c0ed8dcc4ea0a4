// kern_prefix_codes.hip -- kern_prefix.h's kernels for 8-bit pages.
#include "kern_prefix.h"

namespace fgpt {

namespace {
template <int HD>
void launch_hd(hipStream_t s, const paged::PrefixArgs& x, bool qf, int32_t kt, bool pm, bool sm) {
  using namespace paged;
  if (kt == FG_I8 && qf) launch_prefix_m<HD, true, FG_I8>(s, x, pm, sm);
  else if (kt == FG_I8) launch_prefix_m<HD, false, FG_I8>(s, x, pm, sm);
  else if (qf) launch_prefix_m<HD, true, FG_E4M3>(s, x, pm, sm);
  else launch_prefix_m<HD, false, FG_E4M3>(s, x, pm, sm);
}
}  // namespace

void launch_prefix_codes(hipStream_t s, const paged::PrefixArgs& x, int32_t hd, bool qf, int32_t kt, bool pm, bool sm) {
  if (hd == 128) launch_hd<128>(s, x, qf, kt, pm, sm);
  else launch_hd<64>(s, x, qf, kt, pm, sm);
}

}  // namespace fgpt
