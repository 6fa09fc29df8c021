"""Which memory the entry points for any number of new tokens accept (csrc/capi_rows.cpp), on the CPU: its host side over a HIP
runtime of stubs with two allocations on each of two devices. Every pointer that a call follows is looked up, so none to host
memory or to another device's reaches a kernel; calls with good ones reach it."""
import os
import subprocess

import build as mlxr_build

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <string>
#include <vector>
#include "batch.h"
#include "model.h"

#define CHECK(x) do { if (!(x)) { printf("line %d: %s (%s)\n", __LINE__, #x, mlxr::last.c_str()); exit(1); } } while (0)

namespace mlxr {
std::string last;
int launched = 0;
int set_error(int code, const std::string& msg) { last = msg; return code; }
size_t paged_reserve_work(const PagedKV&, int) { return 256; }
size_t paged_attention_rows_work(const PagedKV&, int, int, int) { return 256; }
hipError_t launch_paged_reserve(const ReserveArgs&, hipStream_t) { launched++; return hipSuccess; }
hipError_t launch_paged_append_rows(const AppendRowsArgs&, hipStream_t) { launched++; return hipSuccess; }
hipError_t launch_paged_attention_rows(const AttnRowsArgs&, hipStream_t) { launched++; return hipSuccess; }
}

// device d has the addresses [(d + 1) << 32, + 1 MiB) and the MiB right behind them, as another allocation
static int count = DEVICES;
static int device_of(uintptr_t a) { return a >> 32 >= 1 && a >> 32 <= 2 && (a & 0xffffffffu) < (2u << 20) ? (int)(a >> 32) - 1 : -1; }
extern "C" {
hipError_t hipGetDeviceCount(int* n) { *n = count; return hipSuccess; }
hipError_t hipGetDevice(int* d) { *d = 0; return hipSuccess; }
hipError_t hipGetLastError() { return hipSuccess; }
const char* hipGetErrorString(hipError_t) { return "stub"; }
hipError_t hipStreamGetDevice(hipStream_t s, hipDevice_t* d) { *d = (int)(uintptr_t)s - 1; return hipSuccess; }
hipError_t hipMemGetAddressRange(hipDeviceptr_t* base, size_t* size, hipDeviceptr_t p) {
    const uintptr_t a = (uintptr_t)p;
    if (device_of(a) < 0) { *base = nullptr; *size = 0; return hipErrorNotFound; }
    *base = (hipDeviceptr_t)(a & ~(uintptr_t)0xfffff);
    *size = 1 << 20;
    return hipSuccess;
}
hipError_t hipPointerGetAttribute(void* out, hipPointer_attribute what, hipDeviceptr_t p) {
    CHECK(what == HIP_POINTER_ATTRIBUTE_DEVICE_ORDINAL);
    *(int*)out = device_of((uintptr_t)p);
    return *(int*)out < 0 ? hipErrorInvalidValue : hipSuccess;
}
}

using namespace mlxr;
static const uintptr_t NEAR = (uintptr_t)1 << 32, FAR = (uintptr_t)2 << 32, HOST = 0x7f0000000000;
static uintptr_t at[32];   // a call's pointers
static void* P(int i) { return (void*)at[i]; }

static mlxr_paged_kv cache(int first) {
    return mlxr_paged_kv{P(first), P(first + 1), (int32_t*)P(first + 2), (int32_t*)P(first + 3), (float*)P(first + 4), (int32_t*)P(first + 5), 4, 2, 128, 128, 2, 2, 128, 0};
}
static int reserve(void* s) {
    const mlxr_paged_kv kv = cache(0);
    return mlxr_k_paged_reserve(&kv, (int32_t*)P(6), (int32_t*)P(7), (int32_t*)P(8), 9, (int32_t*)P(9), (int32_t*)P(10), (int32_t*)P(11), (int32_t*)P(12), (int32_t*)P(13),
                                (int32_t*)P(14), P(15), 256, s);
}
static int append(void* s) {
    const mlxr_paged_kv kv = cache(0);
    return mlxr_k_paged_append_rows(&kv, (float*)P(6), 8 * 128, 9, (int32_t*)P(7), (int32_t*)P(8), (int32_t*)P(9), (float*)P(10), 1.0f, (float*)P(11), (float*)P(12), 4, 128, 0,
                                    1e-6f, P(13), 0, 512, s);
}
static int attention(void* s) {
    const mlxr_paged_kv kv = cache(0);
    return mlxr_k_paged_attention_rows(&kv, (int32_t*)P(6), (int32_t*)P(7), 9, P(8), 0, 512, 4, 0, 0.1f, P(9), 512, P(10), 256, s);
}

int main() {
    // a bit for each pointer that the call does not follow
    struct { const char* name; int (*call)(void*); int n, unused; } calls[] = {{"reserve", reserve, 16, 0x33}, {"append", append, 14, 0x8}, {"attention", attention, 11, 0x30}};
    for (auto& c : calls)
        for (int spread = 0; spread < 3; spread++) {   // in one allocation, in two in turn, at the ends of both
            auto good = [&] {
                for (int i = 0; i < 32; i++) at[i] = spread == 0 ? NEAR + 4096 * i : spread == 1 ? NEAR + 4096 * i + ((i & 1) << 20) : NEAR + (i & 1 ? (2 << 20) - 4096 * (i + 1) : 4096 * i);
            };
            launched = 0;
            good();
            CHECK(c.call(nullptr) == MLXR_OK && launched == 1);
            CHECK(c.call((void*)1) == MLXR_OK && launched == 2);
            CHECK(count == 1 || c.call((void*)2) == MLXR_E_INVALID_ARG);
            for (int i = 0; i < c.n; i++) {
                if (c.unused >> i & 1) continue;
                for (uintptr_t wrong : {HOST, NEAR + (2 << 20), NEAR - 4096, FAR + 4096 * i}) {
                    good();
                    at[i] = wrong;
                    const int before = launched, rc = c.call(nullptr);
                    const bool other = wrong >= FAR && wrong < HOST;
                    if (other && count == 1) continue;   // there is no such memory
                    if (rc != MLXR_E_INVALID_ARG || launched != before) { printf("%s: pointer %d at %zx: %d\n", c.name, i, (size_t)wrong, rc); return 1; }
                }
            }
        }
    puts("ok");
}
"""


def test_every_pointer_is_looked_up(tmp_path):
    flags = [*mlxr_build.FLAGS, "--cuda-host-only"]
    obj = tmp_path / "capi.o"
    subprocess.run([mlxr_build.HIPCC, *flags, "-c", os.path.join(mlxr_build.SRC, "capi_rows.cpp"), "-o", str(obj)], check=True, capture_output=True)
    for devices in (1, 2):
        src, test, exe = tmp_path / "t.cpp", tmp_path / "t.o", tmp_path / f"t{devices}"
        src.write_text(PROGRAM)
        subprocess.run([mlxr_build.HIPCC, *flags, f"-DDEVICES={devices}", "-c", str(src), "-o", str(test)], check=True, capture_output=True)
        subprocess.run(["g++", str(test), str(obj), "-o", str(exe)], check=True)
        r = subprocess.run([str(exe)], capture_output=True, text=True)
        assert r.stdout == "ok\n", r.stdout
