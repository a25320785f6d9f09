"""Launches of the verification of drafts: its host code, linked against a runtime that says how many clusters run at the same time. CTAs
take node after node, so no more are launched than that; and where there are more nodes, they are marked as undecided first, so that those
that are out of question are passed over."""
import shutil
import subprocess

import pytest

from create_llm_by_cupy_b200.ops import build as B

PROGRAM = r"""
#include <cuda_runtime_api.h>
#include <cassert>
#include <cstdio>
#include <map>
#include <mutex>
#include <utility>

static int device = 0, queries = 0, refuse = 0;
static std::map<std::pair<int, const void*>, int> allowed;
static int marked = 0, rows_grid = 0, cluster = 0, clusters = 0, walked = 0;

extern "C" {
cudaError_t cudaGetDevice(int* d) { *d = device; return cudaSuccess; }
cudaError_t cudaGetLastError() { return cudaSuccess; }
const char* cudaGetErrorString(cudaError_t) { return ""; }
cudaError_t cudaFuncSetAttribute(const void* f, cudaFuncAttribute, int v) { allowed[{device, f}] = v; return cudaSuccess; }
// 64 registers a thread; GPCs of 18 SMs (and a rest of 4), a cluster lies within one of them
static int at_once(const cudaLaunchConfig_t* c, int cs) {
  const int by_regs = 65536 / (64 * int(c->blockDim.x)), by_smem = int(227 * 1024 / (c->dynamicSmemBytes + 1024));
  const int per = by_regs < by_smem ? by_regs : by_smem;
  return 8 * (18 * per / cs) + 4 * per / cs;
}
cudaError_t cudaOccupancyMaxActiveClusters(int* n, const void*, const cudaLaunchConfig_t* c) {
  ++queries;
  if (refuse > 0) { --refuse; return cudaErrorInvalidValue; }
  assert(c->numAttrs == 1 && c->attrs[0].id == cudaLaunchAttributeClusterDimension);
  *n = at_once(c, c->attrs[0].val.clusterDim.x);
  return cudaSuccess;
}
cudaError_t cudaLaunchKernelExC(const cudaLaunchConfig_t* c, const void* f, void**) {
  const auto at = allowed.find({device, f});
  if (int(c->dynamicSmemBytes) > (at == allowed.end() ? 48 * 1024 : at->second)) return cudaErrorInvalidValue;
  if (c->blockDim.x == 256) ++marked;
  if (c->blockDim.x == 128) ++walked;
  if (c->blockDim.x == 512) {
    cluster = c->gridDim.x;
    rows_grid = c->gridDim.y;
    for (unsigned i = 0; i < c->numAttrs; ++i)
      if (c->attrs[i].id == cudaLaunchAttributeClusterDimension) assert(int(c->attrs[i].val.clusterDim.x) == cluster);
    clusters = at_once(c, cluster);
  }
  return cudaSuccess;
}
cudaError_t cudaLaunchKernel(const void*, dim3, dim3, void**, size_t, cudaStream_t) { return cudaErrorInvalidValue; }
unsigned __cudaPopCallConfiguration(dim3*, dim3*, size_t*, void*) { return 0; }
void** __cudaRegisterFatBinary(void*) { static void* p; return &p; }
void __cudaRegisterFatBinaryEnd(void**) {}
void __cudaUnregisterFatBinary(void**) {}
void __cudaRegisterFunction(void**, const char*, char*, const char*, int, uint3*, uint3*, dim3*, dim3*, int*) {}
int b200_verify_drafts(const void*, const void*, const void*, const void*, const void*, const void*, void*, void*, void*, void*, int, int,
                       int, int, double, double, cudaStream_t);
}
namespace b200 {
int num_sms() { return 148; }
int* status_ptr() { return nullptr; }
}

static int call(int bf16, int B, int n, int V) {             // addresses that the host code only looks at
  char* m = reinterpret_cast<char*>(4096);
  marked = walked = 0;
  return b200_verify_drafts(m, nullptr, m, m, m, nullptr, m, m, m, m, bf16, B, n, V, 0.7, 0.9, nullptr);
}

int main() {
  refuse = 1;                                                // without an answer: one CTA an SM, and asked again
  assert(call(0, 400, 1, 32000) == 0 && rows_grid == 74 && queries == 1);
  assert(call(0, 400, 1, 32000) == 0 && rows_grid == clusters && queries == 2);
  for (int d : {0, 3})
    for (int bf16 : {0, 1})
      for (int V : {1, 600, 4000, 6144, 10900, 17000, 32000, 60001, 140000, 385024})
        for (int B : {1, 4, 9, 37, 150, 700})
          for (int n : {1, 2, 16, 33, 64}) {
            device = d;
            assert(call(bf16, B, n, V) == 0 && walked == 1);
            const int rows = B * n, want = rows < clusters ? rows : clusters;
            if (rows_grid != want || marked != (rows > clusters && n > 1)) {
              std::printf("V %d, %d x %d nodes: %d clusters of %d, %d at once, marked %d\n", V, B, n, rows_grid, cluster, clusters, marked);
              return 1;
            }
          }
  assert(call(1, 700, 64, 600) == 0);
  const int before = queries;                                // an answer is kept
  for (int i = 0; i < 5; ++i) assert(call(1, 700, 64, 600) == 0);
  assert(queries == before);
  return 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="no host compiler")
def test_no_more_clusters_than_run_at_once(tmp_path):
    B.build()
    src, exe = tmp_path / "launch.cpp", tmp_path / "launch"
    src.write_text(PROGRAM)
    obj = B.OUT_DIR / B.OBJ_DIR_NAME / "verify_drafts.o"
    subprocess.run(["g++", "-std=c++17", "-O1", "-UNDEBUG", "-pthread", "-I", str(B.Path(B._nvcc()).resolve().parent.parent / "include"),
                    str(src), str(obj), "-o", str(exe)], check=True)
    run = subprocess.run([str(exe)], timeout=60, capture_output=True, text=True)
    assert run.returncode == 0, run.stdout + run.stderr
