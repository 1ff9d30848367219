"""The serving operators' scratch: calls with it are captured and replayed, and those that cannot get it say so or take the form without."""
import ctypes as C
import subprocess

import pytest

torch = pytest.importorskip("torch")
import serving_util as u  # noqa: E402
from test_gpu_gemm_w4 import check, problem, reference  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,n,k,dtype,a_dtype", [(100, 300, 512, "bf16", "i8"), (70, 4097, 256, "f16", "i8"), (1040, 2050, 512, "bf16", "bf16"), (1040, 2048, 512, "f16", "f16"),
                                                 (20, 300, 512, "bf16", "bf16")])
def test_captured_products_replay(dev, pkg, m, n, k, dtype, a_dtype):
    """Rows widened, weights made first with and without a C of whole vectors, and neither; replayed on other inputs."""
    code = u.codes(pkg.capi)
    a, a_scales, w, scales, z = problem(5, dtype, a_dtype, m, n, k, 64, True)
    c = torch.zeros((m, n), dtype=u.TORCH[dtype], device=u.GPU)

    def run():
        dev.gemm_w4(code[dtype], m, n, k, 64, u.ptr(a), u.ptr(w), u.ptr(scales), u.ptr(c), a_dtype=code[a_dtype], a_scales=u.ptr(a_scales), w_zeros=u.ptr(z),
                    stream=u.stream())

    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
        run()
    for seed in (6, 7):
        for old, new in zip((a, a_scales, w, scales, z), problem(seed, dtype, a_dtype, m, n, k, 64, True)):
            if old is not None:
                old.copy_(new)
        c.zero_()
        graph.replay()
        torch.cuda.synchronize()
        replayed = c.clone()
        run()
        assert torch.equal(c.view(torch.int16), replayed.view(torch.int16))
        check(c, *reference(a, a_scales, w, scales, z, 64), dtype, m)
    assert dev.status() == 0
    del graph


@pytest.mark.parametrize("held", ["bf16", "i8"])
@pytest.mark.parametrize("news", [(1, 1), (4, 1), (70, 1)])
def test_captured_steps_replay(dev, pkg, held, news):
    """Append and attention, few rows and chunks, replayed while the sequences grow."""
    cache = u.Paged(pkg, 51, [(new, 900) for new in news], 2, 128, 16, "bf16", held, junk=0.0)
    q = u.normal(u.gen(52), (cache.tokens, 8, 128)).bfloat16()
    k, v = (u.normal(u.gen(53 + i), (cache.tokens, 2, 128)).bfloat16() for i in range(2))
    o = torch.zeros_like(q)
    view, batch = cache.view(), cache.batch()

    def run():
        dev.kv_page_append(view, batch, pkg.capi.BF16, u.ptr(k), u.ptr(v), stream=u.stream())
        dev.attention_paged(view, batch, pkg.capi.BF16, 8, u.ptr(q), u.ptr(o), stream=u.stream())

    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for lens in ((200, 100), (201, 101), (900, 899)):
        cache.lens.copy_(torch.tensor(lens, dtype=torch.int32))
        cache.seqs = [(new, n) for new, n in zip(news, lens)]
        o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert dev.status() == 0
        want = cache.attend(q)
        assert (o.double() - want).norm() <= 6e-3 * want.norm()
    del graph


NO_SCRATCH = """
#define TSM100_SCRATCH_LIMIT 0
#include "ops_serving.cuh"
#include "ops_w4.cuh"
using namespace tsm100;
template int32_t ops::gemm_w4_typed<__nv_bfloat16>(std::string*, const tsm100_gemm_w4_desc*, const uint8_t*, const w4::Params&, cudaStream_t);
template int32_t ops::gemm_w4_typed<__half>(std::string*, const tsm100_gemm_w4_desc*, const uint8_t*, const w4::Params&, cudaStream_t);
extern "C" int32_t attention_paged(const tsm100_paged_kv* kv, const tsm100_paged_batch* b, const tsm100_attention_paged_desc* d, const void* q, void* o, uint32_t* status,
                                   void* s, char* msg) {
  std::string err;
  const int32_t st = ops::attention_paged(&err, kv, b, d, q, o, status, s);
  std::strncpy(msg, err.c_str(), 199);
  return st;
}
extern "C" int32_t gemm_w4(const tsm100_gemm_w4_desc* d, const void* a, const float* a_scales, const uint8_t* w, const void* w_scales, const uint8_t* zeros, void* c,
                           uint32_t* status, void* s, char* msg) {
  std::string err;
  auto never = [](const tsm100_gemm_desc*, const void*, const void*, void*) { return TSM100_ERR_RUNTIME; };
  const int32_t st = ops::gemm_w4(&err, d, a, a_scales, w, w_scales, zeros, c, status, s, never);
  std::strncpy(msg, err.c_str(), 199);
  return st;
}
"""


@pytest.fixture(scope="module")
def without(tmp_path_factory, pkg):
    """The operators, built so that none of them gets scratch."""
    src = tmp_path_factory.mktemp("no_scratch_serving") / "no_scratch.cu"
    src.write_text(NO_SCRATCH)
    out = src.with_suffix(".so")
    b = pkg.build
    subprocess.run([b.nvcc(), "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-O3", "-split-compile=0", "--expt-relaxed-constexpr", "-w",
                    "-shared", "-Xcompiler", "-fPIC", f"-I{b.CSRC}", f"-I{b.INCLUDE}", "-cudart", "static", "-o", str(out), str(src)], check=True)
    return C.CDLL(str(out))


def address(t):
    return C.c_void_p(u.ptr(t) or None)


@pytest.mark.parametrize("new", [1, 60])
def test_attention_without_scratch_is_refused(pkg, without, new):
    cache = u.Paged(pkg, 54, [(new, 300)], 2, 64, 16, "bf16", "i8")
    q = u.normal(u.gen(55), (new, 4, 64)).bfloat16()
    o, status, msg = torch.full_like(q, 5.0), torch.zeros(1, dtype=torch.int32, device=u.GPU), C.create_string_buffer(200)
    st = without.attention_paged(C.byref(cache.view().desc), C.byref(cache.batch().desc), C.byref(pkg.capi.AttentionPagedDesc(pkg.capi.BF16, 4)), address(q), address(o),
                                 address(status), C.c_void_p(u.stream()), msg)
    torch.cuda.synchronize()
    assert st == pkg.capi.ERR_MEMORY and b"no device memory" in msg.value
    assert (o == 5).all() and int(status[0]) == 0


@pytest.mark.parametrize("m,n,k,a_dtype,st", [(100, 300, 512, "i8", 3), (1040, 2050, 512, "bf16", 0), (20, 300, 512, "i8", 0)])
def test_products_without_scratch(pkg, without, m, n, k, a_dtype, st):
    """More than 64 rows in 8 bits are refused; more than 1024 in 16 make their weights tile by tile; the others need none."""
    code = u.codes(pkg.capi)
    a, a_scales, w, scales, z = problem(8, "bf16", a_dtype, m, n, k, 64, True)
    c, status, msg = torch.full((m, n), 5.0, dtype=torch.bfloat16, device=u.GPU), torch.zeros(1, dtype=torch.int32, device=u.GPU), C.create_string_buffer(200)
    desc = pkg.capi.GemmW4Desc(code["bf16"], code[a_dtype], 64, m, n, k)
    assert st == without.gemm_w4(C.byref(desc), address(a), address(a_scales), address(w), address(scales), address(z), address(c), address(status), C.c_void_p(u.stream()), msg)
    torch.cuda.synchronize()
    assert int(status[0]) == 0
    if st:
        assert st == pkg.capi.ERR_MEMORY and b"no device memory" in msg.value and (c == 5).all()
    else:
        check(c, *reference(a, a_scales, w, scales, z, 64), "bf16", m)
