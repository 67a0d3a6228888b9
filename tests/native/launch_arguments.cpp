// Keeps the second kernel argument of the last launch, of which the test says how many bytes it has.  Loaded with
// RTLD_GLOBAL before fake_hip.cpp's library, to whose hipLaunchKernel (`next`, set by the test) it passes every launch on.
#include <cstddef>
#include <cstdint>
#include <cstring>

struct dim3 { uint32_t x, y, z; };

extern "C" {
int (*next)(const void*, dim3, dim3, void**, size_t, void*) = nullptr;
size_t second_argument_bytes = 0;
char second_argument[256];

int hipLaunchKernel(const void* f, dim3 grid, dim3 block, void** arguments, size_t shared, void* stream) {
    if (second_argument_bytes <= sizeof second_argument) memcpy(second_argument, arguments[1], second_argument_bytes);
    return next(f, grid, block, arguments, shared, stream);
}
}
