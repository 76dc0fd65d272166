// fp16 build of the 8-bit row quantiser (namespace svdq::hf): the bf16 source compiled with the 16-bit type switched.
#define SVDQ_F16 1
#include "quantize_w8a8.cu"
