"""CPU test of the training operators' C entry points when host memory has run out: an error code and
a message, no exception. A small host program makes every ``operator new`` fail during a call; the
calls are refused before any launch."""

import os
import subprocess

import genie_tk._lib as L

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include <dlfcn.h>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <new>
#include "genie_tk_b200.h"

static bool failing = false;
void* operator new(size_t n) {
  void* p = failing ? nullptr : std::malloc(n ? n : 1);
  if (!p) throw std::bad_alloc();
  return p;
}
void operator delete(void* p) noexcept { std::free(p); }
void operator delete(void* p, size_t) noexcept { std::free(p); }

template <typename F>
F find(void* lib, const char* name) {
  F f = reinterpret_cast<F>(dlsym(lib, name));
  if (!f) std::exit(3);
  return f;
}

int main(int, char** argv) {
  void* lib = dlopen(argv[1], RTLD_NOW);
  if (!lib) return 2;
  auto last = find<decltype(&gtk_last_error_string)>(lib, "gtk_last_error_string");
  auto ln = find<decltype(&gtk_layernorm_forward)>(lib, "gtk_layernorm_forward");
  auto lnb = find<decltype(&gtk_layernorm_backward)>(lib, "gtk_layernorm_backward");
  auto norm = find<decltype(&gtk_grad_norm)>(lib, "gtk_grad_norm");
  auto clip = find<decltype(&gtk_clip_grad_norm)>(lib, "gtk_clip_grad_norm");
  auto emb = find<decltype(&gtk_embedding_forward)>(lib, "gtk_embedding_forward");
  auto embb = find<decltype(&gtk_embedding_backward)>(lib, "gtk_embedding_backward");
  void* p = reinterpret_cast<void*>(1 << 20);
  float* f = static_cast<float*>(p);
  const void* grads[2] = {p, p};
  const int64_t numel[2] = {4, 4};
  const int types[2] = {GTK_F32, GTK_F32}, bad[2] = {9, 9};
  for (int round = 0; round < 2; ++round) {
    failing = round == 0;
    int rc[9], i = 0;
    bool said[9];
    auto note = [&](int code) {
      const char* m = last();
      said[i] = m && std::strstr(m, round == 0 ? "memory" : "o");
      if (round == 1 && m && std::strstr(m, "out of host memory")) said[i] = false;
      rc[i++] = code;
    };
    note(ln(p, nullptr, GTK_F32, p, p, GTK_F32, p, f, f, 0, 8, 1e-5f, nullptr));
    note(ln(p, nullptr, 7, p, p, GTK_F32, p, f, f, 4, 8, 1e-5f, nullptr));
    note(lnb(p, nullptr, p, nullptr, GTK_F32, p, GTK_F32, f, f, p, p, p, p, 1, 4, 8, nullptr));
    note(norm(grads, numel, bad, 2, GTK_NORM_2, f, p, 1 << 20, nullptr));
    note(clip(grads, nullptr, numel, types, nullptr, 2, GTK_NORM_2, 1.0, f, p, 1 << 20, nullptr));
    note(clip(grads, nullptr, numel, types, nullptr, 2, GTK_NORM_2, -1.0, f, p, 1 << 20, nullptr));
    note(emb(p, 16, p, GTK_F32, p, 4, 10, 8, 1.f, nullptr, nullptr));
    note(embb(p, GTK_F32, p, 32, p, GTK_F32, 4, 10, 8, 1.f, 10, p, 1 << 20, nullptr, nullptr));
    note(embb(p, GTK_F32, p, 32, p, GTK_F32, 4, 10, 8, 1.f, -1, p, 16, nullptr, nullptr));
    failing = false;
    for (int k = 0; k < i; ++k) {
      std::printf("%d %d\n", rc[k], said[k]);
      if (rc[k] >= 0 || !said[k]) return 1;
    }
  }
  return 0;
}
"""


def test_no_host_memory_is_an_error_code(tmp_path):
    L.load()
    src, exe = tmp_path / "host.cpp", tmp_path / "host"
    src.write_text(PROGRAM)
    # -rdynamic: the library's allocations go through this program's operator new
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    subprocess.run(["g++", "-std=c++17", "-O1", "-rdynamic", "-I", os.path.join(REPO, "include"), "-I",
                    os.path.join(cuda, "include"), str(src), "-o", str(exe), "-ldl"], check=True, timeout=300)
    r = subprocess.run([str(exe), L.LIB_PATH], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, (r.returncode, r.stdout, r.stderr)
    assert len(r.stdout.splitlines()) == 18
