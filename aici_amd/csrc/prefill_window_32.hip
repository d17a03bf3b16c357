// Windowed prefill over caches of 32-token blocks.
#include "prefill_window.h"

namespace hipattn {

void launch_window_images_32(const WindowParams &p, int waves, int dtype, hipStream_t stream) {
  launch_window_images<32>(p, waves, dtype, stream);
}

}  // namespace hipattn
