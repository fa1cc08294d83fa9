// Stands in for the HIP runtime on a machine without a GPU: the library's host code runs, its launches are written down
// and nothing is executed.  Loaded (globally) before libwino_amd.so, so that these definitions are the ones it finds.
// Kept of a launch: the kernel's name, the grid, and the arguments of the tiled products, the first bytes of which are a
// TileArgs each (csrc/tile_gemm.hpp).
#include <cxxabi.h>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <map>
#include <string>

namespace {
struct dim3 { unsigned x, y, z; };
std::map<const void*, std::string>& names() { static std::map<const void*, std::string> m; return m; }
std::string& text() { static std::string t; return t; }
struct { dim3 grid, block; size_t lds; void* stream; } pending;
constexpr int kTileArgs = 136;                          // sizeof(TileArgs)

std::string demangled(std::string name) {
    // _Float16 as the half of older mangling, which every demangler knows
    for (size_t at; (at = name.find("DF16_")) != std::string::npos;) name.replace(at, 5, "Dh");
    int status = 0;
    char* d = abi::__cxa_demangle(name.c_str(), nullptr, nullptr, &status);
    std::string s = d && status == 0 ? d : name;
    std::free(d);
    return s;
}
void write_argument(const void* p) {
    char hex[3];
    text() += ' ';
    for (int i = 0; i < kTileArgs; ++i) {
        std::snprintf(hex, sizeof hex, "%02x", static_cast<const unsigned char*>(p)[i]);
        text() += hex;
    }
}
}  // namespace

extern "C" {
void** __hipRegisterFatBinary(const void*) { static void* handle; return &handle; }
void __hipUnregisterFatBinary(void**) {}
void __hipRegisterVar(void**, void*, char*, char*, int, size_t, int, int) {}
void __hipRegisterFunction(void**, const void* host, char*, const char* device, unsigned, void*, void*, void*, void*, int*) { names()[host] = demangled(device); }
int __hipPushCallConfiguration(dim3 grid, dim3 block, size_t lds, void* stream) { pending = {grid, block, lds, stream}; return 0; }
int __hipPopCallConfiguration(dim3* grid, dim3* block, size_t* lds, void** stream) {
    *grid = pending.grid; *block = pending.block; *lds = pending.lds; *stream = pending.stream;
    return 0;
}
int hipGetDevice(int* d) { *d = 0; return 0; }
int hipGetLastError() { return 0; }
int hipDeviceGetAttribute(int* v, int, int) { *v = 256; return 0; }
int hipFuncSetAttribute(const void*, int, int) { return 0; }

int hipLaunchKernel(const void* host, dim3 grid, dim3 block, void** args, size_t, void*) {
    const std::string& name = names()[host];
    char line[96];
    std::snprintf(line, sizeof line, "%u %u %u %u", grid.x, grid.y, grid.z, block.x);
    text() += name + "|" + line + "|";
    if (name.find("tile_gemm_kernel") != std::string::npos) write_argument(args[0]);
    if (name.find("ce_gradients_kernel") != std::string::npos) { write_argument(args[2]); write_argument(args[5]); }
    text() += '\n';
    return 0;
}
const char* recorded() { return text().c_str(); }
void forget() { text().clear(); }
}
