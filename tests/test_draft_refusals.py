"""What the 4-bit matrices and the verification of drafts refuse, without a GPU: tensors that have shapes, types and a device but no
memory, and a library that must not be asked to launch; and the library's own checks of sizes."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import qwen_engine_amd  # noqa: F401
from qwen_engine_amd.kernels import build, ops

F, B, U8, I32 = torch.float32, torch.bfloat16, torch.uint8, torch.int32


class Launched(Exception):
    pass


class NoLaunch:
    def qe_verify_drafts_workspace_bytes(self, *a):
        return 16

    def qe_gemm_mxfp4_workspace_bytes(self, *a):
        return 0

    def __getattr__(self, name):
        def call(*a):
            raise Launched(name)
        return call


@pytest.fixture
def fake(monkeypatch):
    monkeypatch.setattr(ops, "load_library", lambda: NoLaunch())
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "is_available", lambda: False)      # (else a tensor without memory on cuda:1 asks for that device)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0)
    monkeypatch.setattr(torch.Tensor, "data_ptr", lambda t: 4096)
    with FakeTensorMode():
        yield lambda *s, dtype=F, device="cuda:0": torch.empty(*s, dtype=dtype, device=device)


def mat(t, N, K, device="cuda:0"):
    return ops.MxFp4(t(N, (K + 31) // 32 * 16, dtype=U8, device=device), t(N, (K + 31) // 32, dtype=U8, device=device), K)


def place(monkeypatch, **at):
    """Tensors with the given numbers of elements lie at the given places, all others far from them."""
    at = {int(k[1:]): v for k, v in at.items()}
    monkeypatch.setattr(torch.Tensor, "data_ptr", lambda t: at.get(t.numel(), (1 << 40) + (id(t) << 16)))


def refused(call, *words):
    with pytest.raises(ops.KernelError) as e:
        call()
    for w in words:
        assert w in str(e.value), str(e.value)


def test_quantize(fake):
    t = fake
    with pytest.raises(Launched):
        ops.mxfp4_quantize(t(3, 40))
    refused(lambda: ops.mxfp4_quantize(t(3, 40, dtype=torch.float16)), "element type")
    refused(lambda: ops.mxfp4_quantize(t(3, 40, device="cpu")), "not on the GPU")
    refused(lambda: ops.mxfp4_quantize(t(40)), "shape")
    refused(lambda: ops.mxfp4_quantize(t(3, 4, 32)), "shape")
    refused(lambda: ops.mxfp4_quantize(t(40, 3).T), "contiguous")
    refused(lambda: ops.mxfp4_quantize(t(3, 0)), "no numbers")
    refused(lambda: ops.mxfp4_quantize(t(3, 40, device="cuda:1")), "current device")


def test_values(fake):
    t = fake
    with pytest.raises(Launched):
        ops.mxfp4_values(mat(t, 3, 40))
    refused(lambda: ops.mxfp4_values(t(3, 40)), "no 4-bit matrix")
    refused(lambda: ops.mxfp4_values(mat(t, 3, 40), torch.float16), "element type")
    refused(lambda: ops.mxfp4_values(mat(t, 3, 40)._replace(columns=70)), "shape")
    refused(lambda: ops.mxfp4_values(mat(t, 3, 40)._replace(columns=0)), "columns")
    refused(lambda: ops.mxfp4_values(mat(t, 3, 40)._replace(scales=t(3, 3, dtype=U8))), "shape")
    refused(lambda: ops.mxfp4_values(mat(t, 3, 40)._replace(scales=t(2, 2, dtype=U8))), "shape")
    refused(lambda: ops.mxfp4_values(mat(t, 3, 40)._replace(scales=t(3, 2, dtype=U8, device="cuda:1"))), "expected cuda:0")
    refused(lambda: ops.mxfp4_values(mat(t, 3, 40)._replace(codes=t(3, 32, dtype=torch.int8))), "element type")
    refused(lambda: ops.mxfp4_values(mat(t, 3, 40, "cuda:1")), "current device")


def test_codes_at_an_odd_place(fake, monkeypatch):
    monkeypatch.setattr(torch.Tensor, "data_ptr", lambda t: 4104)
    refused(lambda: ops.mxfp4_values(mat(fake, 3, 40)), "16-byte")
    refused(lambda: ops.gemm_mxfp4(fake(2, 40), mat(fake, 3, 40)), "16-byte")


def test_gemm(fake):
    t = fake
    w = mat(t, 6, 40)
    for x in (t(2, 40), t(2, 40, dtype=B), mat(t, 2, 40)):
        with pytest.raises(Launched):
            ops.gemm_mxfp4(x, w)
    refused(lambda: ops.gemm_mxfp4(t(2, 41), w), "columns")
    refused(lambda: ops.gemm_mxfp4(mat(t, 2, 64), w), "columns")      # (as many blocks, other columns)
    refused(lambda: ops.gemm_mxfp4(t(2, 40, dtype=torch.float16), w), "element type")
    refused(lambda: ops.gemm_mxfp4(t(40, 2).T, w), "contiguous")
    refused(lambda: ops.gemm_mxfp4(t(2, 40), t(6, 40)), "no 4-bit matrix")
    refused(lambda: ops.gemm_mxfp4(t(2, 40), mat(t, 6, 40, "cuda:1")), "expected cuda:0")
    refused(lambda: ops.gemm_mxfp4(t(2, 40, device="cuda:1"), mat(t, 6, 40, "cuda:1")), "current device")
    refused(lambda: ops.gemm_mxfp4(t(2, 40), mat(t, 0, 40)), "no rows")
    refused(lambda: ops.gemm_mxfp4(t(2, 40), w, t(5)), "bias")
    refused(lambda: ops.gemm_mxfp4(t(2, 40), w, t(6, dtype=B)), "bias")
    refused(lambda: ops.gemm_mxfp4(t(2, 40), w, out_dtype=torch.float16), "result")
    refused(lambda: ops.gemm_mxfp4(t(2, 40), w, out=t(2, 5)), "out")
    refused(lambda: ops.gemm_mxfp4(t(2, 40), w, out=t(2, 6, dtype=B)), "out")
    refused(lambda: ops.gemm_mxfp4(t(2, 40), w, out=t(6, 2).T), "out")
    refused(lambda: ops.gemm_mxfp4(t(2, 40), w, epilogue=ops.EPI_RESIDUAL), "stream")
    refused(lambda: ops.gemm_mxfp4(t(2, 40), w, out=t(2, 6, dtype=B), epilogue=ops.EPI_RESIDUAL), "out")
    refused(lambda: ops.gemm_mxfp4(t(2, 40), mat(t, 7, 40), epilogue=ops.EPI_SILU_MUL), "odd")
    refused(lambda: ops.gemm_mxfp4(t(2, 40), w, out=t(2, 6), epilogue=ops.EPI_SILU_MUL), "out")
    for e in (ops.EPI_PARTIAL, ops.EPI_SILU_MUL_IL, ops.EPI_GELU, 9):
        refused(lambda: ops.gemm_mxfp4(t(2, 40), w, epilogue=e), "epilogue")


def test_type_of_the_stream(fake, monkeypatch):
    """A product that is added into the 32-bit stream has no other type, whatever the type of its rows is."""
    t = fake
    place(monkeypatch, n18=4096)
    for x in (t(3, 40), t(3, 40, dtype=B)):
        refused(lambda: ops.gemm_mxfp4(x, mat(t, 6, 40), out_dtype=B, out=t(3, 6), epilogue=ops.EPI_RESIDUAL), "stream")
        for same in (None, F):
            with pytest.raises(Launched):
                ops.gemm_mxfp4(x, mat(t, 6, 40), out_dtype=same, out=t(3, 6), epilogue=ops.EPI_RESIDUAL)


def test_results_over_operands(fake, monkeypatch):
    t = fake
    x, w = t(2, 64), mat(t, 64, 64)
    place(monkeypatch, n128=4096)                              # x and out: the same 128 numbers
    refused(lambda: ops.gemm_mxfp4(x, w, out=t(2, 64)), "over an operand")
    x, w, out = t(3, 64), mat(t, 64, 64), t(3, 64, dtype=B)
    place(monkeypatch, n192=4096)
    refused(lambda: ops.gemm_mxfp4(x, w, out_dtype=B, out=out), "over an operand")
    place(monkeypatch, n192=4096, n2048=4096 + 368)            # (out is 384 bytes; the codes begin 16 before its end)
    refused(lambda: ops.gemm_mxfp4(mat(t, 3, 64), mat(t, 64, 64), out=out), "over an operand")
    place(monkeypatch, n192=4096, n2048=4096 + 384)            # behind it
    with pytest.raises(Launched):
        ops.gemm_mxfp4(mat(t, 3, 64), mat(t, 64, 64), out=out)
    good = dict(logits=t(7, 50), first=t(4, dtype=I32), drafts=t(4, dtype=I32), draft_logits=None, temperature=t(3), accept_uniform=t(4),
                draw_uniform=t(3))
    place(monkeypatch, n7=4096, n4=4096 + 24)                  # tokens, and the drafts at its last element
    refused(lambda: ops.verify_drafts(**good, tokens=t(7, dtype=I32)), "over an operand")
    place(monkeypatch, n3=4096)                                # accepted, and the temperatures
    refused(lambda: ops.verify_drafts(**good, accepted=t(3, dtype=I32)), "over an operand")


def test_verify(fake):
    t = fake
    good = dict(logits=t(7, 50), first=t(4, dtype=I32), drafts=t(4, dtype=I32), draft_logits=t(4, 50), temperature=t(3),
                accept_uniform=t(4), draw_uniform=t(3))
    with pytest.raises(Launched):
        ops.verify_drafts(**good)
    with pytest.raises(Launched):
        ops.verify_drafts(**dict(good, draft_logits=None))
    for name, bad in (("logits", t(7, 50, dtype=B)), ("logits", t(350)), ("logits", t(7, 0)), ("first", t(4, dtype=torch.int64)),
                      ("first", t(0, dtype=I32)), ("first", t(9, dtype=I32)), ("drafts", t(5, dtype=I32)), ("drafts", t(4, dtype=torch.int64)),
                      ("draft_logits", t(4, 51)), ("draft_logits", t(3, 50)), ("draft_logits", t(50, 4).T), ("temperature", t(4)),
                      ("accept_uniform", t(3)), ("accept_uniform", t(4, dtype=torch.float64)), ("draw_uniform", t(4)),
                      ("draw_uniform", t(3, device="cpu")), ("first", t(4, dtype=I32, device="cuda:1"))):
        refused(lambda: ops.verify_drafts(**dict(good, **{name: bad})))
    refused(lambda: ops.verify_drafts(**good, tokens=t(6, dtype=I32)), "tokens")
    refused(lambda: ops.verify_drafts(**good, accepted=t(3)), "accepted")
    there = {k: t(*v.shape, dtype=v.dtype, device="cuda:1") for k, v in good.items()}
    refused(lambda: ops.verify_drafts(**there), "current device")


def test_the_librarys_own_checks():
    """Sizes and places that no kernel takes come back as an error before anything is launched (there is no GPU to launch on)."""
    lib = ctypes.CDLL(str(build.library_path()))
    lib.qe_last_error.restype = ctypes.c_char_p
    vp, i = ctypes.c_void_p, ctypes.c_int
    p = vp(4096)

    def refused(rc, word):
        assert rc == -1 and word in lib.qe_last_error().decode(), (rc, lib.qe_last_error())

    for f in (lib.qe_mxfp4_quantize, lib.qe_mxfp4_values):
        refused(f(p, p, p, i(-1), i(32), i(0), None), "sizes")
        refused(f(p, p, p, i(4), i(0), i(0), None), "sizes")
        refused(f(p, p, p, i(4), i(32), i(7), None), "element type")
        refused(f(p, p, p, i(2 ** 31 - 1), i(2 ** 10), i(0), None), "too many")
    refused(lib.qe_mxfp4_quantize(p, vp(4098), p, i(4), i(32), i(0), None), "whole word")

    def gemm(M=2, N=4, K=32, kind=0, out=0, tail=0, x=p, codes=p):
        return lib.qe_gemm_mxfp4(x, p, codes, p, None, p, i(M), i(N), i(K), i(kind), i(out), i(tail), None, ctypes.c_long(0), None)

    refused(gemm(M=-1), "sizes")
    refused(gemm(N=0), "sizes")
    refused(gemm(K=0), "sizes")
    refused(gemm(K=1 << 30), "sizes")
    refused(gemm(kind=3), "form")
    refused(gemm(tail=3), "form")
    refused(gemm(out=5), "element type")
    refused(gemm(out=1, tail=1), "float32")
    refused(gemm(N=5, tail=2), "odd")
    refused(gemm(codes=vp(4104)), "16-byte")
    refused(gemm(kind=2, x=vp(4104)), "16-byte")
    refused(gemm(M=2 ** 31 - 1), "too many")
    refused(gemm(M=100, kind=1), "workspace")
    lib.qe_verify_drafts_workspace_bytes.restype = ctypes.c_long

    def verify(rows=6, V=50, R=2, ws=p, nbytes=1 << 40):
        return lib.qe_verify_drafts(p, p, p, p, p, p, p, p, p, i(rows), i(V), i(R), ws, ctypes.c_long(nbytes), None)

    refused(verify(rows=1), "sizes")
    refused(verify(V=0), "sizes")
    refused(verify(V=1 << 30), "sizes")
    refused(verify(R=-1, rows=0), "sizes")
    refused(verify(rows=70000), "too many")
    refused(verify(ws=None), "workspace")
    refused(verify(nbytes=64), "workspace")
