"""CPU: the C ABI of the serving operators: descriptor layouts, refusals before any launch, calls without work."""
import ctypes
import os
import re

import pytest
import torch

from actalker_amd import _lib, ops

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "actalker_hip.h")
PAIRS = (("ActhRmsNormDesc", _lib.RmsNormDesc), ("ActhGemmFp8Desc", _lib.GemmFp8Desc),
         ("ActhCausalConvDesc", _lib.CausalConvDesc), ("ActhSsmScanDesc", _lib.SsmScanDesc))


@pytest.fixture(params=[torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def lib(request):
    return _lib.load(request.param)


@pytest.mark.parametrize("name,cls", PAIRS)
def test_layouts(name, cls):
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), open(HEADER).read(), flags=re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    want = []
    for decl in filter(None, (d.strip() for d in body.split(";"))):
        kind = ctypes.c_void_p if "*" in decl else _lib.c_ll if "long long" in decl else \
            _lib.c_float if decl.startswith("float") else _lib.c_int
        want += [(re.search(r"(\w+)\s*$", part).group(1), kind) for part in decl.split(",")]
    assert want == [tuple(f) for f in cls._fields_]


def made(cls, **kw):
    d = cls()
    for k, v in kw.items():
        setattr(d, k, v)
    return d


NORM = dict(x=64, ldx=64, y=64, ldy=64, M=2, C=64, norm=1)
PRODUCT = dict(A=64, lda=64, ascale=64, W=64, ldw=64, wscale=64, C=64, ldc=32, M=2, N=32, K=64)
CONV = dict(x=64, ldx=64, w=64, y=64, ldy=64, T=4, D=64, W=4, nseq=2)
SCAN = dict(u=64, ldu=64, delta=64, ld_delta=64, A=64, B=64, ldb=32, C=64, ldc=32, y=64, ldy=64, T=4, D=64, N=16, G=2, nseq=2)


@pytest.mark.parametrize("fn,cls,good,changes", [
    ("acth_rmsnorm", _lib.RmsNormDesc, NORM, [dict(M=-1), dict(C=0), dict(x=None), dict(y=None), dict(eight=1), dict(ldx=63), dict(ldy=8),
                                              dict(res=64, ldres=8), dict(sum=64, ldsum=8)]),
    ("acth_gemm_fp8", _lib.GemmFp8Desc, PRODUCT, [dict(M=-1), dict(N=0), dict(K=0), dict(A=None), dict(ascale=None), dict(wscale=None),
                                                  dict(C=None), dict(lda=63), dict(ldw=16), dict(ldc=31), dict(R=64, ldr=8)]),
    ("acth_causal_conv", _lib.CausalConvDesc, CONV, [dict(T=-1), dict(D=0), dict(W=1), dict(W=5), dict(nseq=0), dict(nseq=3), dict(x=None), dict(w=None),
                                                     dict(ldx=8), dict(slots=64), dict(state=64, nslots=0), dict(state=64, nslots=1, ld_slot=192),
                                                     dict(state=64, nslots=2, ld_slot=191)]),
    ("acth_ssm_scan", _lib.SsmScanDesc, SCAN, [dict(T=-1), dict(D=0), dict(N=0), dict(N=65), dict(G=0), dict(G=3), dict(nseq=3), dict(u=None), dict(A=None),
                                               dict(B=None), dict(ldu=8), dict(ld_delta=8), dict(ldb=31), dict(ldc=31), dict(z=64, ldz=8), dict(slots=64),
                                               dict(state=64, nslots=2, ld_slot=1023), dict(state=64, nslots=1, ld_slot=1024)]),
])
def test_refusals(lib, fn, cls, good, changes):
    for c in changes:
        assert getattr(lib, fn)(ctypes.byref(made(cls, **{**good, **c})), None) == -1, c
    assert getattr(lib, fn)(None, None) == -1
    assert getattr(lib, fn)(ctypes.byref(made(cls)), None) == 0            # no rows: no pointer is read


def test_scan_workspace(lib):
    size = lib.acth_ssm_scan_workspace_size
    assert size(32, 64, 16, 1, 1, 0) == 0                                  # one short sequence: one walk
    need = size(8192, 2560, 16, 1, 1, 0)
    assert need > 0 and need % 4 == 0
    d = made(_lib.SsmScanDesc, **{**SCAN, "T": 8192, "D": 2560, "ldu": 2560, "ld_delta": 2560, "ldy": 2560, "G": 1, "nseq": 1})
    assert lib.acth_ssm_scan(ctypes.byref(d), None) == -1                   # a long one without its workspace
    d.ws, d.ws_bytes = 64, need - 1
    assert lib.acth_ssm_scan(ctypes.byref(d), None) == -1
    for bad in ((0, 64, 16, 1, 1, 0), (64, 64, 65, 1, 1, 0), (64, 64, 16, 3, 1, 0), (64, 64, 16, 1, 0, 1)):
        assert size(*bad) == 0


def test_cpu_tensors_are_refused():
    x, g = torch.zeros(4, 64, dtype=torch.bfloat16), torch.ones(64)
    q, s = torch.zeros(4, 64, dtype=ops.FP8), torch.ones(4, 1)
    for f in (lambda: ops.rmsnorm(x, g), lambda: ops.rmsnorm_fp8(x, g), lambda: ops.quant_fp8(x), lambda: ops.gemm_fp8(q, s, q, s),
              lambda: ops.causal_conv(x, torch.zeros(64, 4)), lambda: ops.ssm_scan(x, x, torch.zeros(64, 16), x[:, :16], x[:, :16])):
        with pytest.raises(_lib.ActhError, match="device tensor"):
            f()


@pytest.mark.parametrize("N,K", [(1, 1), (128, 128), (130, 200), (257, 96)])
def test_pack_fp8(N, K):
    """Codes times scales are within half a step, 2^-4 of the value or 2^-10 of the scale; rows start at multiples of 16."""
    w = torch.randn(N, K, generator=torch.Generator().manual_seed(1))
    q, s = ops.pack_fp8(w)
    assert q.shape == (N, K) and s.shape == (-(-N // 128), -(-K // 128)) and q.stride() == (-(-K // 16) * 16, 1)
    big = s.double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
    err = (q.float().double() * big - w.double()).abs()
    assert (err <= torch.maximum(w.double().abs() * 2.0 ** -4, big * 2.0 ** -10) * (1 + 2.0 ** -20)).all()
    z, sz = ops.pack_fp8(torch.zeros(3, 5))
    assert (z.float() == 0).all() and (sz > 0).all()


def test_operands_with_a_tangent_are_refused():
    """Forward-mode tangents outlive torch.no_grad(); offsets, codes and absent operands carry none."""
    from torch.autograd import forward_ad
    x, ids, q = torch.randn(3, 4), torch.zeros(4, dtype=torch.int32), torch.zeros(3, 4, dtype=ops.FP8)
    with forward_ad.dual_level():
        ops._not_differentiated("op", (x, None, ids, q))
        d = forward_ad.make_dual(x, torch.ones_like(x))
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises(_lib.ActhError, match="forward-mode"):
                ops._not_differentiated("op", (ids, None, d))
        ops._not_differentiated("op", (forward_ad.unpack_dual(d).primal,))
    ops._not_differentiated("op", (x, ids))
    with pytest.raises(_lib.ActhError, match="no backward"):
        ops._not_differentiated("op", (x, x.clone().requires_grad_()))


def test_sequences_of_no_rows():
    """A batch that has run empty: no rows, no sequences, so no slots either, in a pool of any size."""
    none = torch.zeros(0, dtype=torch.int32)
    for pool in (0, 3):
        got = ops._sequences("op", 0, 0, None, none, none.bool(), torch.zeros(pool, 2, 4))
        assert got[3:] == (0, pool)
    assert ops._sequences("op", 0, 1, None, None, None, None)[3] == 1        # one empty sequence
    for T, nb in ((5, 0), (0, -1), (5, -5), (5, 2)):
        with pytest.raises(_lib.ActhError):
            ops._sequences("op", T, nb, None, None, None, None)
    with pytest.raises(_lib.ActhError):
        ops._sequences("op", 0, 0, None, torch.zeros(1, dtype=torch.int32), None, torch.zeros(2, 2, 4))
