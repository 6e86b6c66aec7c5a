"""encode_fn (csrc/tcgen05.cuh), the driver's function that makes tensor maps: compiled for the CPU against a fake of the lookup, since it is about several threads that need it first."""
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pegainfer_b200", "csrc")

FAKE = r"""
#include <atomic>
#include <chrono>
#include <cstdio>
#include <thread>
#include <vector>
typedef int (*EncodeTiledFn)(int);
enum cudaError_t { cudaSuccess = 0 };
enum cudaDriverEntryPointQueryResult { cudaDriverEntryPointSuccess = 0 };
enum { cudaEnableDefault = 0 };
static std::atomic<int> lookups{0};
static int encode(int v) { return v + 1; }
static cudaError_t cudaGetDriverEntryPoint(const char*, void** p, unsigned long long, cudaDriverEntryPointQueryResult* r) {
  ++lookups;
  std::this_thread::sleep_for(std::chrono::milliseconds(200));
  *p = reinterpret_cast<void*>(encode);
  *r = cudaDriverEntryPointSuccess;
  return cudaSuccess;
}
@@
int main() {
  std::atomic<int> started{0}, good{0};
  std::vector<std::thread> threads;
  for (int i = 0; i < 8; ++i)
    threads.emplace_back([&] {
      ++started;
      while (started < 8) {
      }
      EncodeTiledFn fn = encode_fn();
      if (fn && fn(1) == 2) ++good;
    });
  for (auto& t : threads) t.join();
  printf("%d threads have it, %d lookups\n", good.load(), lookups.load());
  return 0;
}
"""


def test_threads_that_make_their_first_tensor_map_together(tmp_path):
    text = open(os.path.join(CSRC, "tcgen05.cuh")).read()
    at = text.index("inline EncodeTiledFn encode_fn()")
    src = tmp_path / "a.cpp"
    src.write_text(FAKE.replace("@@", text[at:text.index("\n}\n", at) + 3]))
    subprocess.run(["g++", "-std=c++17", "-O1", "-pthread", "-o", str(tmp_path / "a"), str(src)], check=True)
    run = subprocess.run([str(tmp_path / "a")], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0 and run.stdout == "8 threads have it, 1 lookups\n", run.stdout
