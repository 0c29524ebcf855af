"""What launchExpertLayer asks of the HIP runtime, call by call, with a runtime of the test's own under the library (no GPU):
limits of dynamic LDS, which belong to a kernel and not to a call, and the stream's counter when its clearing fails."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

RUNTIME = r"""
#include <stddef.h>
#include <stdlib.h>

typedef struct { unsigned x, y, z; } dim3;

enum { MOST = 256 };
static const void* kernels[MOST];
static int limits[MOST], count, error;
int launches, fail_at = -1, lowered, beyond, held;
const void* launched[MOST];

static int index_of(const void* f)
{
    for (int i = 0; i < count; i++)
        if (kernels[i] == f) return i;
    kernels[count] = f;
    limits[count] = 64 * 1024;
    return count++;
}

static struct { dim3 grid, block; size_t lds; void* s; } given;
int __hipPushCallConfiguration(dim3 grid, dim3 block, size_t lds, void* s)
{
    given.grid = grid, given.block = block, given.lds = lds, given.s = s;
    return 0;
}
int __hipPopCallConfiguration(dim3* grid, dim3* block, size_t* lds, void** s)
{
    *grid = given.grid, *block = given.block, *lds = given.lds, *s = given.s;
    return 0;
}
int hipGetDevice(int* d) { return *d = 0; }
int hipDeviceGetAttribute(int* v, int attribute, int d) { *v = 256; return 0; }
int hipStreamIsCapturing(void* s, int* status) { return *status = 0; }
int hipMalloc(void** p, size_t n) { held++; *p = malloc(n); return 0; }
int hipFree(void* p) { held--; free(p); return 0; }
int hipGetLastError(void) { int e = error; error = 0; return e; }
const char* hipGetErrorString(int e) { return "the test's"; }
int hipFuncSetAttribute(const void* f, int attribute, int value)
{
    int i = index_of(f);
    lowered += value < limits[i];
    limits[i] = value;
    return 0;
}
int hipLaunchKernel(const void* f, dim3 grid, dim3 block, void** args, size_t lds, void* s)
{
    beyond += (int)lds > limits[index_of(f)];
    launched[launches % MOST] = f;
    return error = launches++ == fail_at ? 1 : 0;
}
"""

HEAD = r"""
import ctypes as C, importlib, sys
R = C.CDLL(sys.argv[1], mode=C.RTLD_GLOBAL)
sys.path.insert(0, sys.argv[2])
P = importlib.import_module("3dmaker_amd")
L = P.lib()
number = lambda name: C.c_int.in_dll(R, name)

def call(tokens, experts, topk, dim=192, hidden=136, stream=None, **kw):
    route = P.RouteOption(numExperts=experts, topK=topk, scoreType=0, numGroups=1, topGroups=1, groupScore=2, renormalize=1, scale=1.0)
    o = dict(activation=1, gated=0, weightFormat=0, scaleRows=128, dataType=0, routerType=0, strideX=dim, strideOut=dim)
    o.update(kw)
    option = P.ExpertLayerOption(route=route, dim=dim, hidden=hidden, **o)
    at = 1 << 20  # never read: nothing runs
    L.launchExpertLayer(C.byref(option), at, at, None, at, at, at, at, at, tokens, stream)
    return L.tinymlp_last_error_message().decode() if L.tinymlp_last_error() else ""
"""


def run(tmp_path, body):
    source, library = tmp_path / "runtime.c", tmp_path / "runtime.so"
    source.write_text(RUNTIME)
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", str(library), str(source)], check=True)
    r = subprocess.run([sys.executable, "-c", HEAD + body, str(library), ROOT], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr[-2000:]


def test_no_call_lowers_anothers_limit(tmp_path):
    """A thread may have asked for its limit and not yet launched, or have captured a launch, when another call of the same
    kernel with less LDS comes."""
    run(tmp_path, r"""
for tokens, experts, topk, kw in ((64, 8, 2, {}), (40, 8, 2, {}), (33, 8, 2, {}), (64, 1024, 32, dict(dataType=2)), (64, 300, 2, dict(dataType=2)),
                                  (40, 512, 20, dict(dataType=2)), (64, 64, 32, dict(dataType=1)), (9, 64, 32, dict(dataType=1))):
    assert call(tokens, experts, topk, **kw) == ""
assert number("launches").value > 0 and number("beyond").value == 0
assert number("lowered").value == 0, number("lowered").value
""")


def test_a_counter_that_could_not_be_cleared(tmp_path):
    """The call says so, and the next one of that stream clears it."""
    run(tmp_path, r"""
number("fail_at").value = 0
assert "the test's" in call(4, 8, 2)
assert number("launches").value == 1 and number("held").value == 0
assert call(4, 8, 2) == ""
launched = (C.c_void_p * 256).in_dll(R, "launched")
assert number("launches").value == 5 and launched[1] == launched[0]
assert call(4, 8, 2) == ""  # and clears it once
assert number("launches").value == 8 and launched[0] not in launched[2:8]
""")
