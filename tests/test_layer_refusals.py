"""What the linear layer, the query/key norm with rotation and the e4m3 cache refuse, before anything touches a device."""
import pytest
import torch

import kernel_benchmarking_b200 as kb
from kernel_benchmarking_b200 import _build, _lib

N_ERR, SHAPE, ALIGN, OVERLAP = _lib.RL_ERR_NULL_POINTER, _lib.RL_ERR_BAD_SHAPE, _lib.RL_ERR_ALIGNMENT, _lib.RL_ERR_OVERLAP


@pytest.fixture(scope="module")
def lib():
    _build.build()
    return _lib.load()


# addresses only: every refused call ends before a pointer is followed
A = [0x10000000 * (i + 1) for i in range(10)]


FAR = {k: 0x100000000 * (i + 1) for i, k in enumerate(("x", "W", "bias", "res", "y"))}   # for matrices of many megabytes


def passed(rc):
    """The argument checks let the call through: on a machine without a GPU it then fails in the CUDA runtime."""
    return rc <= _lib.RL_ERR_CUDA or rc in (_lib.RL_OK, _lib.RL_ERR_UNSUPPORTED_ARCH)


no_gpu = pytest.mark.skipif(torch.cuda.is_available(), reason="made-up addresses: an accepted call would run")


def call_linear(lib, x=A[0], W=A[1], bias=A[2], res=A[3], y=A[4], M=128, N=128, K=64, ldx=64, ldw=64, ldr=128, ldy=128, act=0,
                ws=A[5], ws_bytes=1 << 30, variant=0):
    return lib.rl_linear_bf16(_lib.LINEAR_ARGS.pack(*(p or 0 for p in (x, W, bias, res, y, ws)), M, N, K, ldx, ldw, ldr, ldy, act, variant,
                                                    ws_bytes), None)


@pytest.mark.parametrize("rc,kw", [
    (N_ERR, dict(x=None)), (N_ERR, dict(W=None)), (N_ERR, dict(y=None)),
    (SHAPE, dict(M=0)), (SHAPE, dict(N=0)), (SHAPE, dict(K=0)), (SHAPE, dict(M=2 ** 31)), (SHAPE, dict(ws_bytes=-1)), (SHAPE, dict(ldx=56)), (SHAPE, dict(ldw=56)),
    (SHAPE, dict(ldy=120)), (SHAPE, dict(ldr=127)),
    (ALIGN, dict(K=60)), (ALIGN, dict(ldx=68)), (ALIGN, dict(ldw=68)), (ALIGN, dict(x=A[0] + 8)), (ALIGN, dict(bias=A[2] + 8)),
    (ALIGN, dict(ldy=130)), (ALIGN, dict(y=A[4] + 2)), (ALIGN, dict(res=A[3] + 1)),
    (_lib.RL_ERR_BAD_ACTIVATION, dict(act=5)), (_lib.RL_ERR_BAD_ACTIVATION, dict(act=-1)),
    (_lib.RL_ERR_BAD_VARIANT, dict(variant=20)),
    (_lib.RL_ERR_WORKSPACE, dict(M=4096, N=4096, K=4096, ws=None, ldx=4096, ldw=4096, ldr=4096, ldy=4096, **FAR)),
    (_lib.RL_ERR_WORKSPACE, dict(M=4096, N=4096, K=4096, ws_bytes=256, ldx=4096, ldw=4096, ldr=4096, ldy=4096, **FAR)),
    (OVERLAP, dict(y=A[0])), (OVERLAP, dict(y=A[1] + 1024)), (OVERLAP, dict(bias=A[4] + 128 * 128 * 2 - 16)),
    (OVERLAP, dict(res=A[4] + 256)),                 # the residual one row ahead of y
    (OVERLAP, dict(res=A[4], ldr=136)),              # the same start, other rows
])
def test_linear_refuses(lib, rc, kw):
    assert call_linear(lib, **kw) == rc


# (made-up matrices of 4096 x 4096, 32 MiB each, a gigabyte and more apart)
BIG = dict(M=4096, N=4096, K=4096, ldx=4096, ldw=4096, ldr=4096, ldy=4096, **FAR)


@pytest.mark.parametrize("rc,ws", [(ALIGN, 0x10000000004), (ALIGN, 0x10000000008), (OVERLAP, FAR["y"] + 4096 * 8192 - 16),
                                   (OVERLAP, FAR["x"]), (OVERLAP, FAR["W"] - 16), (OVERLAP, FAR["bias"]), (OVERLAP, FAR["res"])])
def test_linear_refuses_workspaces(lib, rc, ws):
    """The kernels store into the workspace 16 bytes at a time: a slice of one that starts elsewhere would fault."""
    nbytes = lib.rl_linear_workspace_bytes(4096, 4096, 4096)
    assert nbytes > 0
    assert call_linear(lib, ws=ws, ws_bytes=nbytes, **BIG) == rc


@no_gpu
def test_linear_accepts_an_aligned_workspace(lib):
    assert passed(call_linear(lib, ws=0x10000000010, ws_bytes=lib.rl_linear_workspace_bytes(4096, 4096, 4096), **BIG))


@no_gpu
def test_linear_accepts(lib):
    assert passed(call_linear(lib))
    assert passed(call_linear(lib, res=A[4]))                                  # the residual is y itself
    assert passed(call_linear(lib, res=A[4] + 256, ldr=256, ldy=256))          # y and the residual side by side in one matrix
    assert passed(call_linear(lib, res=A[3] + 2, ldr=129))                     # rows of the residual need no alignment
    assert passed(call_linear(lib, M=16, ldy=129, y=A[4] + 2))                 # nor those of y for small M
    assert passed(call_linear(lib, bias=None, res=None, ldr=0))
    assert passed(call_linear(lib, ws=None, ws_bytes=0))                       # few tiles need no workspace


def test_linear_workspace_bytes(lib):
    f = lib.rl_linear_workspace_bytes
    assert f(0, 8, 8) == f(8, 0, 8) == f(8, 8, 0) == 0
    for M in (1, 16, 64):
        assert f(M, 4096, 4096) == f(M, 57344, 8192) == 0
    assert f(333, 1000, 1144) == f(128, 4096, 4096) == f(512, 4096, 4096) == 0
    assert f(8192, 4096, 4096) == lib.rl_workspace_bytes(8192, 4096, 4096, 0)
    assert 0 < f(8192, 28672, 8192) < lib.rl_workspace_bytes(8192, 28672, 8192, 0)   # no folded copy of x


def call_qk(lib, q=A[0], k=A[1], gq=A[2], gk=A[3], table=A[4], pos=A[5], p64=1, qo=A[6], ko=A[7], T=64, Hq=8, Hk=2, D=64, rot=64,
            P=128, ldt=64, qt=512, qh=64, kt=128, kh=64, qot=512, qoh=64, kot=128, koh=64, inter=0):
    return lib.rl_qk_norm_rope_bf16(_lib.QK_NORM_ROPE_ARGS.pack(
        *(p or 0 for p in (q, k, gq, gk, table, pos, qo, ko)), T, Hq, Hk, D, rot, P, ldt, qt, qh, kt, kh, qot, qoh, kot, koh, p64,
        inter, 1e-6), None)


@pytest.mark.parametrize("rc,kw", [
    (N_ERR, dict(q=None)), (N_ERR, dict(k=None)), (N_ERR, dict(table=None)), (N_ERR, dict(pos=None)), (N_ERR, dict(qo=None)),
    (N_ERR, dict(ko=None)),
    (SHAPE, dict(T=0)), (SHAPE, dict(Hq=0)), (SHAPE, dict(Hk=0)), (SHAPE, dict(D=264)), (SHAPE, dict(rot=0)), (SHAPE, dict(rot=80)),
    (SHAPE, dict(P=-1)), (SHAPE, dict(T=2 ** 31)), (SHAPE, dict(P=2 ** 32)), (SHAPE, dict(ldt=60)), (SHAPE, dict(qh=-64)),
    (ALIGN, dict(D=60, rot=48)), (ALIGN, dict(rot=56)), (ALIGN, dict(rot=60, inter=1)), (ALIGN, dict(qt=516)),
    (ALIGN, dict(koh=68)), (ALIGN, dict(ldt=66)), (ALIGN, dict(q=A[0] + 8)), (ALIGN, dict(gk=A[3] + 2)),
    (ALIGN, dict(pos=A[5] + 4)), (ALIGN, dict(pos=A[5] + 2, p64=0)),
    (OVERLAP, dict(qo=A[1])), (OVERLAP, dict(ko=A[0] + 1024)), (OVERLAP, dict(qo=A[0] + 128)), (OVERLAP, dict(ko=A[6])),
    (OVERLAP, dict(qot=448)),                        # rows of the output run into each other
    (OVERLAP, dict(qoh=32)), (OVERLAP, dict(qot=0)),
    (OVERLAP, dict(qo=A[4])), (OVERLAP, dict(ko=A[5])),
    (OVERLAP, dict(qo=A[0], qoh=64, qot=512, q=A[0], qh=512, qt=64)),   # in place, but transposed
])
def test_qk_norm_rope_refuses(lib, rc, kw):
    assert call_qk(lib, **kw) == rc


@no_gpu
def test_qk_norm_rope_accepts(lib):
    assert passed(call_qk(lib))
    assert passed(call_qk(lib, qo=A[0], ko=A[1]))                                          # in place
    wide = dict(qt=768, kt=768, q=A[0], k=A[0] + 512 * 2)                                  # q, k, v in one projection's rows
    assert passed(call_qk(lib, **wide))
    assert passed(call_qk(lib, **wide, qo=A[0], ko=A[0] + 512 * 2, qot=768, kot=768))      # in place there
    assert call_qk(lib, **wide, qo=A[0], ko=A[0] + 448 * 2, qot=768, kot=768) == OVERLAP   # k's output over the last query head
    assert passed(call_qk(lib, **wide, qo=A[6], ko=A[0] + 640 * 2, kot=768))               # k's output where v stands
    assert passed(call_qk(lib, qt=64, qh=64 * 64, gq=None, gk=None, inter=1, rot=8, p64=0))   # heads outside
    assert passed(call_qk(lib, qt=0, kt=0))                                                # one token for every position


def call_write(lib, k=A[0], v=A[1], slots=A[2], s64=1, kc=A[3], ks=A[4], vc=A[5], vs=A[6], T=64, H=8, D=64, pages=32, page=16,
               kt=512, kh=64, vt=512, vh=64, cp=8192, co=512, ch=64, sp=128, so=8, sh=1):
    return lib.rl_kv_cache_write_e4m3(_lib.KV_CACHE_WRITE_ARGS.pack(
        *(p or 0 for p in (kc, vc, ks, vs)), pages, page, H, D, cp, co, ch, sp, so, sh, *(p or 0 for p in (k, v, slots)), T, kt, kh,
        vt, vh, s64), None)


@pytest.mark.parametrize("rc,kw", [
    (N_ERR, dict(k=None)), (N_ERR, dict(v=None)), (N_ERR, dict(slots=None)), (N_ERR, dict(kc=None)), (N_ERR, dict(vs=None)),
    (SHAPE, dict(T=0)), (SHAPE, dict(H=0)), (SHAPE, dict(D=264)), (SHAPE, dict(page=0)), (SHAPE, dict(pages=-1)), (SHAPE, dict(pages=2 ** 32 + 1)), (SHAPE, dict(T=2 ** 32 + 1)),
    (SHAPE, dict(kt=-512)), (SHAPE, dict(cp=-8192)),
    (ALIGN, dict(D=60)), (ALIGN, dict(kt=516)), (ALIGN, dict(vh=68)), (ALIGN, dict(co=516)), (ALIGN, dict(k=A[0] + 8)),
    (ALIGN, dict(kc=A[3] + 4)), (ALIGN, dict(ks=A[4] + 2)), (ALIGN, dict(slots=A[2] + 4)),
    (OVERLAP, dict(vc=A[3])), (OVERLAP, dict(vs=A[4])), (OVERLAP, dict(vc=A[3] + 8192)), (OVERLAP, dict(ks=A[3] + 64)),
    (OVERLAP, dict(kc=A[0] + 512)), (OVERLAP, dict(vs=A[2])), (OVERLAP, dict(co=256)), (OVERLAP, dict(sp=0)),
])
def test_kv_cache_write_refuses(lib, rc, kw):
    assert call_write(lib, **kw) == rc


@no_gpu
def test_kv_cache_write_accepts(lib):
    assert passed(call_write(lib))
    assert passed(call_write(lib, vc=A[3] + 8192, cp=16384))                       # keys' and values' pages in turn
    assert passed(call_write(lib, vc=A[3] + 512, co=1024, cp=16384))               # keys and values of a token side by side
    assert passed(call_write(lib, vc=A[3] + 64, ch=128, co=1024, cp=16384))        # ... of a head
    assert passed(call_write(lib, co=64, ch=64 * 16, so=1, sh=16))                 # heads outside the places of a page


def call_read(lib, kc=A[0], ks=A[1], vc=A[2], vs=A[3], table=A[4], cu=A[5], ko=A[6], vo=A[7], total=64, zero=0, B=4, most=8, ldp=8,
              H=8, D=64, pages=32, page=16, cp=8192, co=512, ch=64, sp=128, so=8, sh=1, kt=512, kh=64, vt=512, vh=64):
    return lib.rl_kv_cache_read_e4m3(_lib.KV_CACHE_READ_ARGS.pack(
        *(p or 0 for p in (kc, vc, ks, vs)), pages, page, H, D, cp, co, ch, sp, so, sh, *(p or 0 for p in (table, cu, ko, vo)), total,
        zero, B, most, ldp, kt, kh, vt, vh), None)


@pytest.mark.parametrize("rc,kw", [
    (N_ERR, dict(kc=None)), (N_ERR, dict(vs=None)), (N_ERR, dict(table=None)), (N_ERR, dict(cu=None)), (N_ERR, dict(ko=None)),
    (SHAPE, dict(total=0)), (SHAPE, dict(B=-1)), (SHAPE, dict(most=-1)), (SHAPE, dict(D=264)), (SHAPE, dict(vh=-8)),
    (ALIGN, dict(D=60)), (ALIGN, dict(ko=A[6] + 8)), (ALIGN, dict(kt=516)), (ALIGN, dict(cu=A[5] + 2)), (ALIGN, dict(table=A[4] + 1)),
    (OVERLAP, dict(vo=A[6])), (OVERLAP, dict(vo=A[6] + 512)), (OVERLAP, dict(ko=A[0])), (OVERLAP, dict(vo=A[5])),
    (OVERLAP, dict(ko=A[4])), (OVERLAP, dict(kt=256)), (OVERLAP, dict(vt=0)),
])
def test_kv_cache_read_refuses(lib, rc, kw):
    assert call_read(lib, **kw) == rc


@no_gpu
def test_kv_cache_read_accepts(lib):
    assert passed(call_read(lib))
    assert passed(call_read(lib, B=0, table=None))
    assert passed(call_read(lib, vo=A[6] + 1024, kt=1024, vt=1024))    # keys and values of a token side by side


@no_gpu
def test_shared_memory_is_told_apart_from_interleaving(lib):
    """Random strided outputs around each other: any shared byte is refused (never the other way round), and most
    interleavings that share none are accepted."""
    import itertools
    import random
    r = random.Random(5)
    D, seen = 16, {True: 0, False: 0}
    refused_apart = 0
    for _ in range(4000):
        T, Hq, Hk = r.randint(1, 4), r.randint(1, 4), r.randint(1, 4)
        # strides of one parent array, heads or tokens outside, with gaps; the two outputs as windows of it, or as they come
        if r.random() < 0.5:
            inner = 16 * r.randint(1, 2)
            outer = inner * r.randint(max(Hq, Hk), 10)
            st = dict(qot=outer, qoh=inner, kot=outer, koh=inner)
        else:
            st = dict(qot=16 * r.randint(0, 8), qoh=16 * r.randint(0, 8), kot=16 * r.randint(0, 8), koh=16 * r.randint(0, 8))
        shift = 16 * r.randint(-40, 40)

        def covered(base, H, t, h):
            return [base + a * t + b * h + d for a, b, d in itertools.product(range(T), range(H), range(0, D, 8))]

        q, k = covered(0, Hq, st["qot"], st["qoh"]), covered(shift, Hk, st["kot"], st["koh"])
        shares = len(set(q)) < len(q) or len(set(k)) < len(k) or bool(set(q) & set(k))
        rc = call_qk(lib, qo=A[6], ko=A[6] + 2 * shift, T=T, Hq=Hq, Hk=Hk, D=D, rot=16, ldt=16, **st)
        seen[shares] += 1
        if shares:
            assert rc == OVERLAP, (T, Hq, Hk, st, shift)
        else:
            refused_apart += rc == OVERLAP
            assert rc == OVERLAP or passed(rc)
    assert min(seen.values()) > 300 and refused_apart < 0.2 * seen[False]


def test_argument_structures(lib):
    """The packed formats are the header's structures: pointers and 64-bit integers, no padding."""
    assert _lib.LINEAR_ARGS.size == 8 * 16 and _lib.QK_NORM_ROPE_ARGS.size == 8 * 26 and _lib.KV_CACHE_WRITE_ARGS.size == 8 * 23 and _lib.KV_CACHE_READ_ARGS.size == 8 * 27
    for f in (lib.rl_linear_bf16, lib.rl_qk_norm_rope_bf16, lib.rl_kv_cache_write_e4m3, lib.rl_kv_cache_read_e4m3):
        assert f(None, None) == N_ERR


def test_new_error_strings(lib):
    for code in (_lib.RL_ERR_BAD_INDEX, OVERLAP, _lib.RL_ERR_BAD_ACTIVATION):
        assert _lib.error_string(code) != "unknown error code"
    with pytest.raises(ValueError):
        _lib.check(OVERLAP, "x")
    with pytest.raises(RuntimeError):
        _lib.check(_lib.RL_ERR_BAD_INDEX, "x")


def test_no_cpu_path():
    x, W = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(8, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        kb.linear(x, W)
    q = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        kb.qk_norm_rope(q, q, None, None, torch.zeros(8, 64), torch.zeros(4, dtype=torch.int64))
    c, s = torch.zeros(2, 16, 2, 64, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.zeros(2, 16, 2)
    with pytest.raises(ValueError, match="CUDA"):
        kb.kv_cache_write(q, q, torch.zeros(4, dtype=torch.int64), c, s, c, s)
    with pytest.raises(ValueError, match="CUDA"):
        kb.kv_cache_read(c, s, c, s, torch.zeros(1, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), 4)
    with pytest.raises(TypeError):
        kb.linear([1], W)
    with pytest.raises(TypeError):
        kb.qk_norm_rope([1], q, None, None, None, None)


def test_rope_table():
    t = kb.rope_table(50000, 16, device="cpu")
    assert t.shape == (50000, 16) and t.dtype == torch.float32
    import math
    for p in (0, 1, 49999):
        for i in range(8):
            angle = p * 10000.0 ** (-2 * i / 16)
            assert abs(t[p, i].item() - math.cos(angle)) <= 2.0 ** -24 + 1e-11
            assert abs(t[p, 8 + i].item() - math.sin(angle)) <= 2.0 ** -24 + 1e-11
    for bad in ((0, 16), (4, 0), (4, 7)):
        with pytest.raises(ValueError):
            kb.rope_table(*bad, device="cpu")
