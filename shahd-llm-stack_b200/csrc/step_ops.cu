// The third translation unit of libshahd_b200.so: operators of a serving step over shared pages that wait for nothing inside their
// kernels (section 4 of shahd_b200.h). They keep no state on a device.
#include "logits.cuh"
#include "norm_rope.cuh"
#include "pages.cuh"
