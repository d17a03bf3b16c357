// Windowed prefill over caches of 8-token blocks.
#include "prefill_window.h"

namespace hipattn {

void launch_window_images_8(const WindowParams &p, int waves, int dtype, hipStream_t stream) {
  launch_window_images<8>(p, waves, dtype, stream);
}

}  // namespace hipattn
