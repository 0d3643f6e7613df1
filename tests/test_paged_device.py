"""The caller's current device after calls of the paged operators on another
one.  Runs without a GPU: a child process puts a stand-in for the CUDA
runtime's device and launch calls before the library."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

FAKE = r"""
#include <stddef.h>
int current, sets, launches, launched_on, major_of[4] = {10, 10, 9, 10}, fail;
int cudaGetDevice(int* d) { *d = current; return 0; }
int cudaSetDevice(int d) { current = d, ++sets; return 0; }
int cudaGetDeviceCount(int* n) { *n = 4; return 0; }
int cudaDeviceGetAttribute(int* v, int what, int d) {
  *v = what == 75 ? major_of[d] : what == 76 ? 0 : 148;  /* major, minor, SMs */
  return 0;
}
static int launch(void) { ++launches, launched_on = current; return fail; }
int cudaLaunchKernel(const void* f) { return launch(); }
int cudaLaunchKernelExC(const void* f) { return launch(); }
int cudaMemsetAsync(void* p, int v, size_t n, void* s) { return launch(); }
int cudaFuncSetAttribute(const void* f, int a, int v) { return 0; }
int cudaGetLastError(void) { return fail; }
static int encode(void) { return 0; }
int cudaGetDriverEntryPoint(const char* name, void** p, unsigned long long flags, int* r) {
  *p = (void*)encode, *r = 0;
  return 0;
}
"""

CHILD = r"""
import ctypes as C, sys
fake = C.CDLL(sys.argv[1], mode=C.RTLD_GLOBAL)
import modelc_b200 as mb
from test_paged import APPEND, ATTENTION, PROMPT, READ, ROPE, SLOTS, _call
L = mb.lib()
var = {n: C.c_int.in_dll(fake, n) for n in ("current", "sets", "launches", "launched_on", "fail")}
heads = dict(head_dim=128, n_kv_heads=2, dtype=2)
calls = {
    "mc_paged_slots": lambda d: _call("mc_paged_slots", SLOTS, d, n_requests=2, n_tokens=4, page_size=64,
                                      table_width=4, n_free_pages=4),
    "mc_rope_table": lambda d: L.mc_rope_table(4096, 32, 10, 1.0, 4096, 4096, d, None),
    "mc_rope": lambda d: _call("mc_rope", ROPE, d, rot=128, n_tokens=4, n_heads=8, n_kv_heads=8, head_dim=128,
                               table_rows=10, q_tok=1024, q_head=128, k_tok=1024, k_head=128),
    "mc_kv4_append": lambda d: _call("mc_kv4_append", APPEND, d, n_pages=9, n_tokens=3, k_tok=256, k_head=128,
                                     v_tok=256, v_head=128, **heads),
    "mc_kv4_read": lambda d: _call("mc_kv4_read", READ, d, n_pages=9, n_tokens=3, **heads),
    "mc_kv4_attention": lambda d: _call("mc_kv4_attention", ATTENTION, d, n_heads=4, n_tokens=3, scale=0.1, n_pages=9,
                                        n_requests=1, table_width=4, q_tok=512, q_head=128,
                                        workspace_bytes=1 << 30, **heads),
    "mc_prompt_attention": lambda d: _call("mc_prompt_attention", PROMPT, d, n_heads=4, n_q=3, n_k=3, scale=0.1,
                                           causal=1, n_sequences=1, q_tok=512, q_head=128, k_tok=256, k_head=128,
                                           v_tok=256, v_head=128, **heads),
    "no keys": lambda d: _call("mc_prompt_attention", PROMPT, d, n_heads=4, n_q=3, scale=0.1, n_sequences=1,
                               q_tok=512, q_head=128, k_tok=256, k_head=128, v_tok=256, v_head=128, **heads),
}
call = calls[sys.argv[2]]
# another device: the launches happen there, and the caller's is current again
assert call(1) == 0 and var["launches"].value > 0 and var["launched_on"].value == 1
assert var["current"].value == 0
# the caller's own device is not set again
var["sets"].value = 0
assert call(0) == 0 and var["launched_on"].value == 0 and var["sets"].value == 0
# an error on the way out
var["fail"].value = 700
assert call(3) == -5 and var["launched_on"].value == 3 and var["current"].value == 0
var["fail"].value = 0
# refused devices
for d in (2, 4, -1, 64):
    assert call(d) in (-1, -5) and var["current"].value == 0
# the size of a workspace needs no device to be current
var["sets"].value = 0
assert L.mc_kv4_attention_workspace(3, 128, 1) > 0 and L.mc_kv4_attention_workspace(3, 128, 2) == 0
assert var["sets"].value == 0 and var["current"].value == 0
print("done")
"""


@pytest.fixture(scope="module")
def fake(tmp_path_factory):
    d = tmp_path_factory.mktemp("runtime")
    src, lib = d / "fake.c", d / "libfake.so"
    src.write_text(FAKE)
    subprocess.run(["gcc", "-shared", "-fPIC", "-w", "-o", str(lib), str(src)], check=True)
    return str(lib)


@pytest.mark.parametrize("name", ["mc_paged_slots", "mc_rope_table", "mc_rope", "mc_kv4_append", "mc_kv4_read",
                                  "mc_kv4_attention", "mc_prompt_attention", "no keys"])
def test_the_current_device_stays(fake, name):
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([ROOT, os.path.join(ROOT, "tests")]))
    r = subprocess.run([sys.executable, "-c", CHILD, fake, name], env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.split() == ["done"], r.stderr[-2000:]
