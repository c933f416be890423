"""Emit and build the per-model shared library.

The reference's code generator writes a self-contained C++17 source whose
exported functions run the model on the CPU (src/codegen.cpp:24-50,
673-1130).  Here the per-model source is a thin C++ shim: it embeds the
graph blob (weights included) with ``.incbin`` and exports the reference's
C ABI names, forwarding every call to the CUDA engine in
libforgetune_b200.so on a model handle it creates on first use.  Only the
host compiler runs per model; the kernels are built once, in-tree.
"""

from __future__ import annotations

import os
import subprocess

from . import build_native
from .build_native import INCLUDE, LIB_DIR, LIB_PATH
from .errors import CompilationError

_TEMPLATE = r'''// Generated by forgetune_b200 -- per-model drop-in for the reference C ABI.
// graph blob: @BLOB_NAME@ (@BLOB_BYTES@ bytes, sha256 @BLOB_SHA@)
#include <cstddef>
#include <cstdint>
#include <mutex>

#include "forgetune_b200.h"

__asm__(
    ".section .rodata\n"
    ".balign 64\n"
    ".local ftb_embedded_blob\n"
    "ftb_embedded_blob:\n"
    ".incbin \"@BLOB_PATH@\"\n"
    ".local ftb_embedded_blob_end\n"
    "ftb_embedded_blob_end:\n"
    ".previous\n");
extern "C" const unsigned char ftb_embedded_blob[];
extern "C" const unsigned char ftb_embedded_blob_end[];

namespace {
std::mutex g_mu;
void* g_model = nullptr;
int g_rc = 0;
int g_policy = -1;
int g_devs[64];
int g_ndev = 0;

void* model() noexcept {
  std::lock_guard<std::mutex> lk(g_mu);
  if (!g_model) {
    g_rc = ftb_model_create(ftb_embedded_blob, (size_t)(ftb_embedded_blob_end - ftb_embedded_blob), &g_model);
    if (g_rc != 0) {
      g_model = nullptr;
      return nullptr;
    }
    if (g_policy >= 0) ftb_model_set_policy(g_model, g_policy);
    if (g_ndev > 0) ftb_model_set_devices(g_model, g_devs, g_ndev);
  }
  return g_model;
}

struct Unload {
  ~Unload() {
    std::lock_guard<std::mutex> lk(g_mu);
    if (g_model) ftb_model_destroy(g_model);
    g_model = nullptr;
  }
} g_unload;
}  // namespace

@RUN_ENTRY@

extern "C" FORGETUNE_EXPORT int forgetune_run_v2(const float* input, size_t input_count, float* output,
                                                 size_t output_count, int64_t batch_size) {
  void* m = model();
  if (!m) return -4;
  return ftb_model_run(m, input, input_count, output, output_count, batch_size, FTB_API_V2);
}

extern "C" FORGETUNE_EXPORT int forgetune_run_v1(const float* input, size_t input_count, float* output,
                                                 size_t output_count) {
  void* m = model();
  if (!m) return -4;
  return ftb_model_run(m, input, input_count, output, output_count, -1, FTB_API_V1);
}

extern "C" FORGETUNE_EXPORT int forgetune_is_dynamic(void) { return @IS_DYNAMIC@; }

extern "C" FORGETUNE_EXPORT int64_t forgetune_max_batch(void) { return @MAX_BATCH@; }

extern "C" FORGETUNE_EXPORT double forgetune_benchmark_kernel(const float* input, size_t input_count,
                                                              float* output, size_t output_count,
                                                              int iters) {
  if (!input || !output || iters <= 0) return -1.0;
  void* m = model();
  if (!m) return -4.0;
  return ftb_model_benchmark(m, input, input_count, output, output_count, iters);
}

extern "C" FORGETUNE_EXPORT size_t forgetune_get_arena_alloc_count(void) {
  void* m = model();
  return m ? ftb_model_counter(m, 0) : 0;
}
extern "C" FORGETUNE_EXPORT size_t forgetune_get_arena_payload_alloc_count(void) {
  void* m = model();
  return m ? ftb_model_counter(m, 1) : 0;
}
extern "C" FORGETUNE_EXPORT size_t forgetune_get_arena_block_insertion_count(void) {
  void* m = model();
  return m ? ftb_model_counter(m, 2) : 0;
}
extern "C" FORGETUNE_EXPORT size_t forgetune_get_process_arena_total_allocations(void) {
  void* m = model();
  return m ? ftb_model_counter(m, 3) : 0;
}
extern "C" FORGETUNE_EXPORT void forgetune_reset_arena_alloc_count(void) {
  void* m = model();
  if (m) ftb_model_reset_counters(m);
}
extern "C" FORGETUNE_EXPORT void forgetune_test_inject_arena_alloc(void) {
  void* m = model();
  if (m) ftb_model_inject_alloc(m);
}

extern "C" FORGETUNE_EXPORT int forgetune_create(void) {
  void* m = model();
  if (!m) return g_rc ? g_rc : -4;
  return ftb_model_prepare(m);
}

extern "C" FORGETUNE_EXPORT void forgetune_destroy(void) {
  std::lock_guard<std::mutex> lk(g_mu);
  if (g_model) ftb_model_destroy(g_model);
  g_model = nullptr;
}

extern "C" FORGETUNE_EXPORT int forgetune_set_devices(const int* device_ids, int n) {
  if (n < 0 || n > 64 || (n > 0 && !device_ids)) return -1;
  {
    std::lock_guard<std::mutex> lk(g_mu);
    for (int i = 0; i < n; ++i) g_devs[i] = device_ids[i];
    g_ndev = n;
  }
  void* m = model();
  if (!m) return -4;
  return ftb_model_set_devices(m, device_ids, n);
}

extern "C" FORGETUNE_EXPORT int forgetune_set_kernel_policy(int policy) {
  {
    std::lock_guard<std::mutex> lk(g_mu);
    g_policy = policy;
  }
  void* m = model();
  if (!m) return -4;
  return ftb_model_set_policy(m, policy);
}

extern "C" FORGETUNE_EXPORT int forgetune_run_v2_device(const float* d_input, size_t input_count, float* d_output,
                                                        size_t output_count, int64_t batch_size,
                                                        void* stream) {
  void* m = model();
  if (!m) return -4;
  return ftb_model_run_device(m, d_input, input_count, d_output, output_count, batch_size, stream);
}

extern "C" FORGETUNE_EXPORT int forgetune_describe(char* buf, size_t cap) {
  void* m = model();
  if (!m) return -4;
  return ftb_model_describe(m, buf, cap);
}
'''

_RUN_DYNAMIC = r'''extern "C" FORGETUNE_EXPORT int forgetune_run(const float* input, size_t input_count, float* output,
                                              size_t output_count, int64_t batch_size) {
  void* m = model();
  if (!m) return -4;
  return ftb_model_run(m, input, input_count, output, output_count, batch_size, FTB_API_RUN);
}'''

_RUN_STATIC = r'''extern "C" FORGETUNE_EXPORT int forgetune_run(const float* input, size_t input_count, float* output,
                                              size_t output_count) {
  void* m = model();
  if (!m) return -4;
  return ftb_model_run(m, input, input_count, output, output_count, 0, FTB_API_RUN);
}'''


def emit_source(blob_path: str, blob_bytes: int, blob_sha: str, dynamic: bool, max_batch: int) -> str:
    """C++ source of the per-model shim for the blob stored at ``blob_path``."""
    if '"' in blob_path or "\\" in blob_path or "\n" in blob_path:
        raise CompilationError("artifact path contains characters the assembler cannot quote: %r" % blob_path)
    src = _TEMPLATE
    for k, v in {
        "@BLOB_NAME@": os.path.basename(blob_path),
        "@BLOB_BYTES@": str(blob_bytes),
        "@BLOB_SHA@": blob_sha,
        "@BLOB_PATH@": blob_path,
        "@IS_DYNAMIC@": "1" if dynamic else "0",
        "@MAX_BATCH@": str(int(max_batch)),
        "@RUN_ENTRY@": _RUN_DYNAMIC if dynamic else _RUN_STATIC,
    }.items():
        src = src.replace(k, v)
    return src


def host_compiler() -> str:
    c = build_native.host_compiler()
    if c:
        return c
    raise CompilationError("no host C++ compiler found (g++, c++ or clang++)")


def compile_shim(cpp_path: str, so_path: str, opt_level: str = "-O2", timeout: int = 300) -> None:
    """g++ the shim into ``so_path`` (atomic replace), linked to the in-tree engine library."""
    if not os.path.isfile(LIB_PATH):
        raise CompilationError("libforgetune_b200.so is not built; run `python -m forgetune_b200.build_native`")
    tmp = so_path + ".tmp%d" % os.getpid()
    cmd = [host_compiler(), "-shared", "-fPIC", "-std=c++17", opt_level, "-Wall", "-Wextra",
           "-fvisibility=hidden", "-I", INCLUDE, "-o", tmp, cpp_path,
           "-L", LIB_DIR, "-lforgetune_b200", "-Wl,-rpath," + LIB_DIR,
           # export only the ABI, never symbols of a statically linked runtime
           "-Wl,--exclude-libs,ALL"]
    try:
        r = subprocess.run(cmd, capture_output=True, text=True, timeout=timeout)
    except subprocess.TimeoutExpired as e:
        raise CompilationError("host compiler timed out after %ds" % timeout, command=cmd) from e
    if r.returncode != 0:
        raise CompilationError("host compiler failed (%d): %s" % (r.returncode, r.stderr[-4000:]),
                               stdout=r.stdout, stderr=r.stderr, command=cmd)
    os.replace(tmp, so_path)
