/* A context and tensors without a device, to see what the ops refuse: a call that is refused says why,
 * one that passes its checks fails at the device (there is none) without a message. */
#include <stdlib.h>

#include "qw_internal.h"

h3_gpu *fake_context(int device, int open) {
    h3_gpu *gpu = calloc(1, sizeof(*gpu));
    gpu->device = device;
    gpu->chain_open = open;
    return gpu;
}
void fake_open(h3_gpu *gpu, int open) { gpu->chain_open = open, gpu->error[0] = 0; }
h3_gpu_tensor *fake_tensor(h3_gpu *gpu, int dtype, size_t elements) {
    h3_gpu_tensor *tensor = calloc(1, sizeof(*tensor));
    tensor->owner = gpu;
    tensor->dtype = (h3_gpu_dtype)dtype;
    tensor->elements = elements;
    return tensor;
}
