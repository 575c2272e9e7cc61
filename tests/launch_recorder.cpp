// The HIP runtime's entry points that the library's launches call, as a recorder: nothing is launched.  Loaded in front of the library with
// global visibility.
#include <stddef.h>
#include <stdint.h>

struct Dim3 {
    uint32_t x, y, z;
};
static int launches, too_large;
static uint64_t workgroups;
static const void* last_kernel;
static thread_local Dim3 config_grid, config_block;
static thread_local size_t config_lds;
static thread_local void* config_stream;

extern "C" {
int hipGetLastError() { return 0; }
int hipLaunchKernel(const void* kernel, Dim3 grid, Dim3 block, void**, size_t, void*) {
    ++launches;
    last_kernel = kernel;
    workgroups += (uint64_t)grid.x * grid.y * grid.z;
    too_large += (uint64_t)grid.x * block.x >= (uint64_t(1) << 32) || grid.y > 65535 || grid.x == 0;
    return 0;
}
int __hipPushCallConfiguration(Dim3 grid, Dim3 block, size_t lds, void* stream) {
    config_grid = grid, config_block = block, config_lds = lds, config_stream = stream;
    return 0;
}
int __hipPopCallConfiguration(Dim3* grid, Dim3* block, size_t* lds, void** stream) {
    *grid = config_grid, *block = config_block, *lds = config_lds, *stream = config_stream;
    return 0;
}
void recorder_reset() { launches = too_large = 0, workgroups = 0, last_kernel = nullptr; }
int recorder_launches() { return launches; }
int recorder_too_large() { return too_large; }  // launches of more threads than the runtime takes
uint64_t recorder_workgroups() { return workgroups; }
const void* recorder_kernel() { return last_kernel; }
}
