"""Attention over pages that cannot get its scratch names the operator that was called, whichever kernel it would have taken."""
import ctypes as C
import subprocess

import pytest

torch = pytest.importorskip("torch")
import serving_util as u  # noqa: E402
from test_gpu_attention_paged_cross import Encoded  # noqa: E402

pytestmark = pytest.mark.gpu

NO_SCRATCH = """
#define TSM100_SCRATCH_LIMIT 0
#include "ops_serving.cuh"
using namespace tsm100;
extern "C" int32_t attend(int32_t cross, const tsm100_paged_kv* kv, const tsm100_paged_batch* b, const tsm100_attention_paged_desc* d, const void* q, void* o, uint32_t* status,
                          void* stream, char* msg) {
  std::string err;
  paged::Params p;
  bool nothing;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int32_t st = ops::attention_paged_args(&err, "args", kv, b, d->dtype, d->heads_q, q, o, status, &p, &nothing);
  if (st == TSM100_OK) st = cross ? ops::attention_cross_launch<__nv_bfloat16, false, 64>(&err, p, q, o, s) : ops::attention_paged_launch<__nv_bfloat16, false, 64>(&err, p, q, o, s);
  std::strncpy(msg, err.c_str(), 199);
  return st;
}
"""


@pytest.fixture(scope="module")
def without(tmp_path_factory, pkg):
    src = tmp_path_factory.mktemp("no_scratch_names") / "no_scratch.cu"
    src.write_text(NO_SCRATCH)
    out = src.with_suffix(".so")
    b = pkg.build
    subprocess.run([b.nvcc(), "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-O1", "-split-compile=0", "--expt-relaxed-constexpr", "-w",
                    "-shared", "-Xcompiler", "-fPIC", f"-I{b.CSRC}", f"-I{b.INCLUDE}", "-cudart", "static", "-o", str(out), str(src)], check=True)
    return C.CDLL(str(out))


@pytest.mark.parametrize("new", [1, 12, 60])
@pytest.mark.parametrize("cross,name", [(0, b"attention_paged: "), (1, b"attention_paged_cross: ")])
def test_the_name(pkg, without, cross, name, new):
    cache = Encoded(pkg, 54, [(new, 300)], 2, 64, 16, "bf16", "bf16")
    q = u.normal(u.gen(55), (new, 4, 64)).bfloat16()
    o, status, msg = torch.full_like(q, 5.0), torch.zeros(1, dtype=torch.int32, device=u.GPU), C.create_string_buffer(200)
    st = without.attend(cross, C.byref(cache.view().desc), C.byref(cache.batch().desc), C.byref(pkg.capi.AttentionPagedDesc(pkg.capi.BF16, 4)), *map(C.c_void_p, (u.ptr(q), u.ptr(o), u.ptr(status))),
                        C.c_void_p(u.stream()), msg)
    torch.cuda.synchronize()
    assert st == pkg.capi.ERR_MEMORY and msg.value.startswith(name) and b"no device memory" in msg.value and (o == 5).all() and int(status[0]) == 0
