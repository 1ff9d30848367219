"""8-bit products of odd rows, cross attention and attention behind a shared prefix that cannot get their scratch say so and touch nothing; products of aligned rows need none."""
import ctypes as C
import subprocess

import pytest

torch = pytest.importorskip("torch")
import serving_util as u  # noqa: E402
from test_gpu_attention_paged_cross import Encoded  # noqa: E402
from test_gpu_attention_paged_prefix import Sharing  # noqa: E402
from test_gpu_gemm_i8 import check, problem, reference  # noqa: E402

pytestmark = pytest.mark.gpu

NO_SCRATCH = """
#define TSM100_SCRATCH_LIMIT 0
#include "ops_i8.cuh"
#include "ops_serving.cuh"
using namespace tsm100;
extern "C" int32_t prefix(const tsm100_paged_kv* kv, const tsm100_paged_batch* b, const tsm100_attention_paged_prefix_desc* d, const void* q, void* o, uint32_t* status, void* s,
                          char* msg) {
  std::string err;
  paged::Params p;
  bool nothing;
  int32_t st = ops::attention_paged_args(&err, "attention_paged_prefix", kv, b, d->dtype, d->heads_q, q, o, status, &p, &nothing);
  ops::PrefixArgs more = {};
  more.prefix = d->prefix_len, more.table = d->prefix;
  p.step.table += d->prefix_len / kv->page_size;
  if (st == TSM100_OK)
    st = ops::attention_prefix_launch<__nv_bfloat16, false, 64>(&err, p, ops::PrefixPlan{false, false, 4}, more, q, o, static_cast<cudaStream_t>(s));
  std::strncpy(msg, err.c_str(), 199);
  return st;
}
extern "C" int32_t cross(const tsm100_paged_kv* kv, const tsm100_paged_batch* b, const tsm100_attention_paged_desc* d, const void* q, void* o, uint32_t* status, void* s, char* msg) {
  std::string err;
  paged::Params p;
  bool nothing;
  int32_t st = ops::attention_paged_args(&err, "attention_paged_cross", kv, b, d->dtype, d->heads_q, q, o, status, &p, &nothing);
  if (st == TSM100_OK) st = ops::attention_cross_launch<__nv_bfloat16, false, 64>(&err, p, q, o, static_cast<cudaStream_t>(s));
  std::strncpy(msg, err.c_str(), 199);
  return st;
}
extern "C" int32_t product(const tsm100_gemm_i8_desc* d, const void* a, const float* a_scales, const void* w, const float* w_scales, void* c, uint32_t* status, void* s, char* msg) {
  std::string err;
  const int32_t st = ops::gemm_i8(&err, d, a, a_scales, w, w_scales, c, status, s);
  std::strncpy(msg, err.c_str(), 199);
  return st;
}
"""


@pytest.fixture(scope="module")
def without(tmp_path_factory, pkg):
    """The operators, built so that none of them gets scratch."""
    src = tmp_path_factory.mktemp("no_scratch_more") / "no_scratch.cu"
    src.write_text(NO_SCRATCH)
    out = src.with_suffix(".so")
    b = pkg.build
    subprocess.run([b.nvcc(), "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-O1", "-split-compile=0", "--expt-relaxed-constexpr", "-w",
                    "-shared", "-Xcompiler", "-fPIC", f"-I{b.CSRC}", f"-I{b.INCLUDE}", "-cudart", "static", "-o", str(out), str(src)], check=True)
    return C.CDLL(str(out))


def address(t):
    return C.c_void_p(u.ptr(t) or None)


@pytest.mark.parametrize("new", [1, 60])
def test_cross_attention(pkg, without, new):
    cache = Encoded(pkg, 54, [(new, 300)], 2, 64, 16, "bf16", "bf16")
    q = u.normal(u.gen(55), (new, 4, 64)).bfloat16()
    o, status, msg = torch.full_like(q, 5.0), torch.zeros(1, dtype=torch.int32, device=u.GPU), C.create_string_buffer(200)
    st = without.cross(C.byref(cache.view().desc), C.byref(cache.batch().desc), C.byref(pkg.capi.AttentionPagedDesc(pkg.capi.BF16, 4)), address(q), address(o),
                       address(status), C.c_void_p(u.stream()), msg)
    torch.cuda.synchronize()
    assert st == pkg.capi.ERR_MEMORY and b"no device memory" in msg.value and (o == 5).all() and int(status[0]) == 0


def test_behind_a_prefix(pkg, without):
    cache = Sharing(pkg, 54, [(1, 30), (2, 40)], 2, 64, 16, "bf16", "bf16", 3)
    q = u.normal(u.gen(55), (3, 4, 64)).bfloat16()
    o, status, msg = torch.full_like(q, 5.0), torch.zeros(1, dtype=torch.int32, device=u.GPU), C.create_string_buffer(200)
    d = pkg.capi.AttentionPagedPrefixDesc(pkg.capi.BF16, 4, 48, u.ptr(cache.prefix))
    st = without.prefix(C.byref(cache.view().desc), C.byref(cache.batch().desc), C.byref(d), address(q), address(o), address(status), C.c_void_p(u.stream()), msg)
    torch.cuda.synchronize()
    assert st == pkg.capi.ERR_MEMORY and b"no device memory" in msg.value and (o == 5).all() and int(status[0]) == 0


@pytest.mark.parametrize("m,n,k", [(3, 100, 501), (300, 400, 512), (3, 100, 512)])
def test_products(pkg, without, m, n, k):
    a, a_scales, w, w_scales = problem(1, m, n, k)
    c, status, msg = torch.full((m, n), 5.0, dtype=torch.bfloat16, device=u.GPU), torch.zeros(1, dtype=torch.int32, device=u.GPU), C.create_string_buffer(200)
    d = pkg.capi.GemmI8Desc(pkg.capi.BF16, m, n, k, 0, 0, 0)
    st = without.product(C.byref(d), address(a), address(a_scales), address(w), address(w_scales), address(c), address(status), C.c_void_p(u.stream()), msg)
    torch.cuda.synchronize()
    if k % 16:
        assert st == pkg.capi.ERR_MEMORY and b"no device memory" in msg.value and (c == 5).all()
    else:
        assert st == pkg.capi.OK
        check(c, reference(a, a_scales, w, w_scales), "bf16")
    assert int(status[0]) == 0
