// launches.cpp -- stands in for the HIP runtime's launch entry points, so that what
// the library launches can be seen without a GPU: every kernel's name, grid, block
// and stream go to a callback, and nothing runs. Loaded with its symbols global
// before the libraries (tests/launches.py), in a process of its own.
#include <cstddef>
#include <cstdint>
#include <string>
#include <unordered_map>
#include <vector>

namespace {

struct Dim3 {  // dim3's layout
    uint32_t x, y, z;
};
struct Config {
    Dim3 grid, block;
    size_t shared;
    void *stream;
};

struct Kernels {
    std::vector<std::string> names;  // "translation unit:mangled name", in order of registration
    std::unordered_map<const void *, int> of;
    int units = 0;
};
Kernels &kernels() {
    static Kernels k;
    return k;
}
thread_local Config config;
void (*on_launch)(const char *, const uint32_t *, const uint32_t *, void *) = nullptr;
int handle;
void *fat_binary = &handle;

}  // namespace

extern "C" {

void **__hipRegisterFatBinary(const void *) {
    ++kernels().units;
    return &fat_binary;
}
void __hipUnregisterFatBinary(void **) {}
void __hipRegisterVar(void **, void *, char *, char *, int, size_t, int, int) {}
void __hipRegisterManagedVar(void *, void **, void *, const char *, size_t, unsigned) {}
void __hipRegisterFunction(void **, const void *host, char *, const char *name, unsigned, void *, void *, void *, void *, int *) {
    Kernels &k = kernels();
    k.of[host] = (int)k.names.size();
    k.names.push_back(std::to_string(k.units) + ":" + name);
}
int __hipPushCallConfiguration(Dim3 grid, Dim3 block, size_t shared, void *stream) {
    config = {grid, block, shared, stream};
    return 0;
}
int __hipPopCallConfiguration(Dim3 *grid, Dim3 *block, size_t *shared, void **stream) {
    *grid = config.grid;
    *block = config.block;
    *shared = config.shared;
    *stream = config.stream;
    return 0;
}
int hipLaunchKernel(const void *kernel, Dim3 grid, Dim3 block, void **, size_t, void *stream) {
    const uint32_t g[3] = {grid.x, grid.y, grid.z}, b[3] = {block.x, block.y, block.z};
    if (on_launch != nullptr) on_launch(kernels().names.at(kernels().of.at(kernel)).c_str(), g, b, stream);
    return 0;
}
int hipGetLastError() { return 0; }

// What the tests call: the callback (null: none), and the kernels that the libraries have.
void launches_to(void (*f)(const char *, const uint32_t *, const uint32_t *, void *)) { on_launch = f; }
int launches_kernels() { return (int)kernels().names.size(); }
const char *launches_kernel(int i) { return kernels().names.at(i).c_str(); }
}
