"""Parts of the 4-bit kernels' device code that are plain C++, compiled for the host and run there (CPU tests)."""
import re
import subprocess

from accy_amd.build import KERNELS

HOST = """
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <vector>
#define __device__
#define __forceinline__ inline
typedef uint32_t u32_t;
"""


def _function(name):
    """The source of a function template of mx4.h, its template line included."""
    text = (KERNELS / "mx4.h").read_text()
    found = re.search(r"^template <[^\n]*>\n__device__ __forceinline__ [\w ]+ " + name + r"\(.*?^}\n", text, re.S | re.M)
    assert found, name
    return found.group(0)


def _run(tmp_path, body):
    source = tmp_path / "host.cpp"
    source.write_text(HOST + body)
    subprocess.run(["g++", "-std=c++17", "-O1", "-w", "-o", str(tmp_path / "host"), str(source)], check=True)
    out = subprocess.run([str(tmp_path / "host")], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0, out.stdout


def test_search_for_later_tokens_stays_in_its_array(tmp_path):
    """A workgroup's threads one after the other, in order and in reverse, over token counts around a thread's and a pass's reach, slots
    of which many are padding and many the same: each token that a later one of its slot follows loses it, and no element
    before or after the array is touched."""
    _run(tmp_path, _function("leave_to_later") + """
template <int TW> int check(unsigned seed) {
  int bad = 0;
  for (int left : {1, 2, TW, TW + 1, 3 * TW, 255, 256, 257, 300, 2049, 2400})
    for (int back = 0; back < 2; ++back) {
      srand(seed + left);
      std::vector<int> slots(left);
      for (int& s : slots) { const int r = rand() % 8; s = r < 3 ? -1 : r == 3 ? -2147483647 - 1 : r == 4 ? 1 << 30 : rand() % (left / 2 + 1); }
      int place[16 + TW + 16];
      for (int& p : place) p = 12345;
      for (int w = 0; w < TW; ++w) place[16 + w] = w < left && slots[w] >= 0 && slots[w] < 1 << 30 ? slots[w] : -1;
      for (int t = 0; t < 256; ++t) leave_to_later<TW>(place + 16, slots.data(), left, back ? 255 - t : t);
      for (int i = 0; i < 16; ++i) bad += place[i] != 12345 || place[16 + TW + i] != 12345;
      for (int w = 0; w < TW; ++w) {
        int want = w < left && slots[w] >= 0 && slots[w] < 1 << 30 ? slots[w] : -1;
        for (int j = w + 1; j < left; ++j) if (want >= 0 && slots[j] == want) want = -1;
        bad += place[16 + w] != want;
      }
    }
  if (bad) printf("TW %d: %d wrong\\n", TW, bad);
  return bad;
}
int main() {
  return (check<1>(1) + check<2>(2) + check<3>(3) + check<4>(4) + check<5>(5) + check<6>(6) + check<7>(7) + check<8>(8) + check<10>(9) + check<21>(10) +
          check<64>(11) + check<128>(12)) != 0;
}
""")
