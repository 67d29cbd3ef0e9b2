"""The linear layer, the query/key norm with rotation and the e4m3 cache against their definitions in 64 bits.

Tolerances, per element, derived from the arithmetic:
  one rounding to bf16            2^-8 |y|   (half a step)
  linear: fp32 sum of K products  (K + 2) 2^-23 sum |x w|, an adder that may cut off counted with a whole step, times the
                                  steepest slope of an activation (gelu 1.13); fast exponential: e^t carries |t| 2^-22 from
                                  its argument and 2^-16 of its own, at |t| <= 88 less than 2^-14 of the result
  norm and rotation               sum of D squares, root, two products, rotation: (D / 2 + 10) 2^-24 of |n_i c| + |n_j s|
  cache                           none: codes, scales and what is read back are exactly rounded
"""
import math

import pytest
import torch

import kernel_benchmarking_b200 as kb

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, E4M3 = torch.bfloat16, torch.float8_e4m3fn
HALF_STEP = 2.0 ** -8
ACTS = [None, "relu", "gelu", "gelu_tanh", "silu"]


def rnd(*shape, seed, scale=1.0):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(BF16)


def done():
    torch.cuda.synchronize()
    kb.check_status()


# ------------------------------------------------------------------ linear

def act64(z, act):
    if act == "relu":
        return z.clamp(min=0)
    if act == "gelu":
        return z * torch.special.erfc(-z / math.sqrt(2)) / 2
    if act == "gelu_tanh":
        return z * torch.sigmoid(math.sqrt(8 / math.pi) * (z + 0.044715 * z ** 3))
    if act == "silu":
        return z * torch.sigmoid(z)
    return z


def check_linear(y, x, W, bias, act, residual):
    xd, Wd = x.double(), W.double()
    z = xd @ Wd.t()
    S = xd.abs() @ Wd.abs().t()
    if bias is not None:
        z = z + bias.double()
        S = S + bias.double().abs()
    a = act64(z, act)
    ref = a if residual is None else a + residual.double()
    tol = HALF_STEP * ref.abs() + 1.2 * (x.shape[1] + 2) * 2.0 ** -23 * S + 2.0 ** -14 * a.abs() + 2.0 ** -22 * ref.abs() + 1e-30
    assert y.shape == ref.shape and y.dtype == BF16
    over = ((y.double() - ref).abs() - tol).max().item()
    assert over <= 0, f"beyond the tolerance by {over}"


def linear_inputs(M, N, K, seed, bias, residual):
    return (rnd(M, K, seed=seed), rnd(N, K, seed=seed + 1, scale=K ** -0.5), rnd(N, seed=seed + 2) if bias else None,
            rnd(M, N, seed=seed + 3) if residual else None)


@pytest.mark.parametrize("M,N,K", [(1, 8, 8), (1, 4096, 4096), (3, 1, 64), (16, 129, 72), (17, 1000, 520), (33, 4104, 1032), (64, 136, 4096),
                                   (65, 8, 8), (65, 77, 64), (128, 256, 64), (129, 520, 328), (300, 1001, 1144), (512, 1024, 4096)])
@pytest.mark.parametrize("act,bias,residual", [(None, False, False), (None, False, True), ("relu", True, False), ("gelu", True, True),
                                               ("gelu_tanh", True, False), ("silu", False, True)])
def test_linear(M, N, K, act, bias, residual):
    x, W, b, r = linear_inputs(M, N, K, M + N + K, bias, residual)
    y = kb.linear(x, W, b, activation=act, residual=r)
    done()
    check_linear(y, x, W, b, act, r)


@pytest.mark.parametrize("M,N,K", [
    (148, 4874, 808), (66, 2110, 1720), (1003, 19, 4464), (40, 14, 5800),    # 64-token tiles, long ring, clusters of 1, 2, 4, 8
    (387, 2845, 528), (83, 4829, 1104), (82, 2305, 3696),                    # 128-token tiles, long ring, clusters of 1, 2, 4
    (971, 1929, 72), (222, 2485, 512), (265, 1948, 4528),                    # 128-token tiles, two CTAs on an SM
    (64, 4097, 112), (64, 4916, 328), (40, 4136, 2176), (40, 10, 1968)])     # 64-token tiles, two CTAs on an SM
@pytest.mark.parametrize("act,bias,residual", [("gelu", True, True), (None, False, False)])
def test_linear_of_few_tiles(M, N, K, act, bias, residual):
    """Every tile, cluster size and ring of the cluster kernel, with ragged last tiles, twice with the same result."""
    x, W, b, r = linear_inputs(M, N, K, 25, bias, residual)
    y = kb.linear(x, W, b, activation=act, residual=r)
    again = kb.linear(x, W, b, activation=act, residual=r)
    done()
    check_linear(y, x, W, b, act, r)
    assert torch.equal(y, again)


@pytest.mark.parametrize("M,N,K", [(4096, 1536, 4096),      # 96 tiles: one round, 22 cut in three
                                   (2048, 5120, 2048),      # a last round cut in four
                                   (8192, 7168, 4096),      # 256 x 512 tiles
                                   (4100, 7176, 4104),      # ... with ragged edges everywhere
                                   (16384, 2048, 512)])
@pytest.mark.parametrize("act,bias,residual", [("gelu", True, True), (None, False, True)])
def test_linear_large(M, N, K, act, bias, residual):
    x, W, b, r = linear_inputs(M, N, K, 5, bias, residual)
    y = kb.linear(x, W, b, activation=act, residual=r)
    whole = kb.linear(x, W, b, activation=act, residual=r, variant="auto_whole")
    again = kb.linear(x, W, b, activation=act, residual=r)
    done()
    check_linear(y, x, W, b, act, r)
    check_linear(whole, x, W, b, act, r)
    assert torch.equal(y, again)


@pytest.mark.parametrize("M,N,K,act,bias,residual", [
    (8192, 4096, 13312, "gelu", True, True),         # 256 tiles of 256 x 512: the last 34 cut in two
    (5800, 5000, 13320, "gelu_tanh", True, True),    # 230, ragged: the last 8 cut in four
    (5800, 5000, 8200, None, False, True),
    (5800, 5000, 9224, "silu", False, False)])
def test_linear_on_wide_tiles(M, N, K, act, bias, residual):
    """K-loops long enough for the 256 x 512 tiles' exposed epilogue, whole and with a last round cut along K; in place."""
    x, W, b, r = linear_inputs(M, N, K, 15, bias, residual)
    whole = kb.linear(x, W, b, activation=act, residual=r, variant="auto_whole")
    y = kb.linear(x, W, b, activation=act, residual=r)
    again = kb.linear(x, W, b, activation=act, residual=r)
    done()
    check_linear(y, x, W, b, act, r)
    check_linear(whole, x, W, b, act, r)
    assert torch.equal(y, again)
    if r is not None:
        kb.linear(x, W, b, activation=act, residual=r, out=r)
        done()
        assert torch.equal(r, y)


@pytest.mark.parametrize("M,N,K,pairs", [(300, 520, 328, False), (2048, 5120, 2048, True), (8192, 7168, 4096, True)])
def test_linear_without_epilogue_is_the_plain_gemm(M, N, K, pairs):
    x, W, _, _ = linear_inputs(M, N, K, 9, False, False)
    y, g = kb.linear(x, W), kb.gemm_nt(x, W)
    done()
    check_linear(y, x, W, None, None, None)
    if pairs:      # the same tiles add the k-blocks in the same order; few tiles are cut along K, which changes the sums' order
        assert torch.equal(y, g)


@pytest.mark.parametrize("M", [1, 40, 200, 4096])
def test_linear_in_place_on_the_residual_and_strided(M):
    N, K = 1032, 264
    x = rnd(M, K + 24, seed=1)[:, 8:8 + K]
    W = rnd(N, 2 * K, seed=2, scale=K ** -0.5)[:, K:]
    stream = rnd(M + 2, N + 40, seed=3)
    keep = stream.clone()
    h = stream[1:1 + M, 16:16 + N]
    y = kb.linear(x, W, activation="silu", residual=h, out=h)
    done()
    assert y.data_ptr() == h.data_ptr()
    check_linear(h, x, W, None, "silu", keep[1:1 + M, 16:16 + N])
    keep[1:1 + M, 16:16 + N] = h
    assert torch.equal(stream, keep)      # nothing around it changed


@pytest.mark.parametrize("M", [5, 200])
def test_linear_residual_with_odd_rows(M):
    N, K = 136, 64
    x, W, b, _ = linear_inputs(M, N, K, 3, True, False)
    wide = rnd(M, N + 3, seed=8)
    for r in (wide[:, :N], wide[:, 3:]):
        y = kb.linear(x, W, b, residual=r)
        done()
        check_linear(y, x, W, b, None, r)
    one_row = rnd(1, N, seed=9).expand(M, N)   # the same row for every token
    y = kb.linear(x, W, b, residual=one_row)
    done()
    check_linear(y, x, W, b, None, one_row)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M", [2, 100])
def test_linear_extreme_values(act, M):
    """Large, tiny and non-finite pre-activations arrive through the bias (x = 0); the residual stays out of the way."""
    N = 64
    vals = [0.0, -0.0, 1e-30, -1e-30, 0.5, -0.5, 5.0, -5.0, 9.0, -9.0, 20.0, -20.0, 90.0, -90.0, 1e4, -1e4, 1e30, -1e30,
            float("inf"), float("nan")]
    b = torch.tensor(vals + [1.0] * (N - len(vals)), device=DEV).to(BF16)
    y = kb.linear(torch.zeros(M, 64, dtype=BF16, device=DEV), rnd(N, 64, seed=1), b, activation=act)
    done()
    ref = act64(b.double(), act).expand(M, N)
    fine = ref.isfinite()
    assert torch.equal(y.double()[~fine].nan_to_num(nan=7.0), ref[~fine].nan_to_num(nan=7.0))
    assert bool(((y.double() - ref)[fine].abs() <= (HALF_STEP + 2.0 ** -14) * ref[fine].abs() + 1e-30).all())


def test_single_rows_with_meaningless_strides():
    """A dimension of one element may have any stride."""
    K, N, D = 64, 72, 64
    x = rnd(K, 1, seed=1).t()                                  # [1, K] with strides (1, 1)
    W, r = rnd(N, K, seed=2), rnd(N, 1, seed=3).t()
    y = kb.linear(x, W, residual=r)
    w1 = kb.linear(rnd(5, K, seed=4), rnd(K, 1, seed=5).t())
    done()
    check_linear(y, x, W, None, None, r)
    check_linear(w1, rnd(5, K, seed=4), rnd(K, 1, seed=5).t(), None, None, None)
    q = rnd(2 * D + 7, seed=6)[:D].as_strided((1, 1, D), (3, 5, 1))
    pos, table = torch.tensor([3], device=DEV), kb.rope_table(8, D, device=DEV)
    yq, yk = kb.qk_norm_rope(q, q, None, None, table, pos)
    one = kb.qk_norm_rope(q, q, None, None, table[3:4].as_strided((1, D), (1, 1)), pos - 3)
    done()
    check_qk(yq, q, None, table, pos, False)
    assert torch.equal(yq, yk) and torch.equal(one[0], yq)
    cache = [torch.zeros(D, dtype=torch.uint8, device=DEV).view(E4M3).as_strided((1, 1, 1, D), (5, 3, 1, 1)) if i % 2 == 0 else
             torch.zeros(1, device=DEV).as_strided((1, 1, 1), (7, 7, 7)) for i in range(4)]
    zero = torch.zeros(1, dtype=torch.int64, device=DEV)
    kb.kv_cache_write(q, q, zero, *cache)
    ko, vo = kb.kv_cache_read(*cache, torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.tensor([0, 1], dtype=torch.int32, device=DEV), 1)
    done()
    check_written(cache, q, q, zero)
    val, sc = quant64(q)
    assert torch.equal(ko.cpu(), (val.float() * sc[..., None]).to(BF16)) and torch.equal(ko, vo)


def test_linear_refusals():
    x, W, b, r = linear_inputs(100, 64, 64, 1, True, True)
    for kw in (dict(activation="tanh"), dict(residual=r[:, :60]), dict(residual=r.float()), dict(out=x), dict(out=r[:, :32]),
               dict(variant="decode"), dict(workspace=torch.zeros(16, device=DEV))):
        with pytest.raises(ValueError):
            kb.linear(x, W, b, **kw)
    for args in ((x, W.float()), (x, W, b[:32]), (x, W, b.float()), (x[:, :60], W[:, :60]), (x, W[:, :32])):
        with pytest.raises(ValueError):
            kb.linear(*args)
    big = linear_inputs(4096, 2048, 4096, 1, False, False)
    with pytest.raises(ValueError, match="workspace"):
        kb.linear(big[0], big[1], workspace=torch.zeros(1024, dtype=torch.uint8, device=DEV))
    flat = torch.zeros(100 * 64 + 64, dtype=BF16, device=DEV)
    with pytest.raises(ValueError, match="shares memory"):
        kb.linear(x, W, residual=flat[64:].view(100, 64), out=flat[:-64].view(100, 64))
    assert kb.linear(x[:0], W).shape == (0, 64) and kb.linear(x, W[:0]).shape == (100, 0)
    done()


def test_linear_workspaces_that_start_anywhere():
    """A slice of a larger buffer serves from any 16-byte boundary; elsewhere, and inside an operand, it is refused."""
    M, N, K = 4096, 1536, 4096   # cuts tiles along K
    x, W, b, r = linear_inputs(M, N, K, 61, True, True)
    want = kb.linear(x, W, b, residual=r)
    n = kb.linear_workspace(M, N, K, x.device).numel()
    assert n > 0
    flat = torch.zeros(n + 64, dtype=torch.uint8, device=DEV)
    for at in (4, 8, 17):
        with pytest.raises(ValueError, match="aligned"):
            kb.linear(x, W, b, residual=r, workspace=flat[at:])
    assert torch.equal(kb.linear(x, W, b, residual=r, workspace=flat[16:]), want)
    big = torch.zeros(n // 2 + M * N, dtype=BF16, device=DEV)
    with pytest.raises(ValueError, match="shares memory"):
        kb.linear(x, W, b, workspace=big.view(torch.uint8), out=big[:M * N].view(M, N))
    done()


@pytest.mark.parametrize("M,N,K", [(8, 2048, 1024), (300, 520, 1024), (4096, 2048, 4096)])
@pytest.mark.parametrize("own", [False, True])
def test_linear_in_two_graphs_at_once(M, N, K, own):
    """Two graphs of the operator, replayed on two streams at once: they share no scratch."""
    graphs = []
    for i in range(2):
        x, W, b, r = linear_inputs(M, N, K, 50 + i, True, True)
        ws = kb.linear_workspace(M, N, K, x.device) if own else None
        want = kb.linear(x, W, b, activation="silu", residual=r, variant="auto_whole")
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = kb.linear(x, W, b, activation="silu", residual=r, workspace=ws, variant="auto_whole")
        graphs.append((g, y, want, (x, W, b, r, ws)))
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for (g, y, _, _), s in zip(graphs, sides):
            with torch.cuda.stream(s):
                g.replay()
    done()
    for g, y, want, _ in graphs:
        assert torch.equal(y, want)


def test_linear_k_split_in_a_graph_and_grown_workspaces():
    """A captured call that cuts tiles along K, replayed after eager calls of other sizes."""
    x, W, b, r = linear_inputs(4096, 1536, 4096, 60, True, True)
    want = kb.linear(x, W, b, residual=r)
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        y = kb.linear(x, W, b, residual=r)
    for (M, N, K) in ((1, 4096, 512), (64, 1000, 1024), (3000, 2048, 1024)):
        kb.linear(*linear_inputs(M, N, K, 61, False, False)[:2])
    for _ in range(3):
        g.replay()
    done()
    assert torch.equal(y, want)


@pytest.mark.parametrize("seed", range(4))
def test_linear_random_shapes(seed):
    """Sizes spread over their logarithms, so over every tile and cluster size of the plan, with every way to call it."""
    import random
    r = random.Random(1000 + seed)
    for i in range(50):
        M, N = int(math.exp(r.uniform(0, math.log(3000)))), int(math.exp(r.uniform(0, math.log(6000))))
        K = 8 * int(math.exp(r.uniform(0, math.log(512))))
        act, s = r.choice(ACTS), 10 * i + 7 * seed
        x, W, b, _ = linear_inputs(M, N, K, s, r.random() < 0.5, False)
        kind = r.choice(["none", "plain", "odd", "in place"])
        res = out = None
        if kind == "plain":
            res = rnd(M, N, seed=s + 5)
        elif kind == "odd":
            res = rnd(M, N + 5, seed=s + 5)[:, 3:3 + N]
        elif kind == "in place":
            res = out = rnd(M, (N + 7) // 8 * 8 + 8, seed=s + 5)[:, :N]
        keep = None if res is None else res.clone()
        y = kb.linear(x, W, b, activation=act, residual=res, out=out, variant=r.choice(["auto", "auto_whole"]))
        torch.cuda.synchronize()
        check_linear(y, x, W, b, act, keep)
    done()


def test_linear_on_a_side_stream():
    x, W, b, r = linear_inputs(33, 1024, 1024, 70, True, True)
    want = kb.linear(x, W, b, residual=r)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        y = kb.linear(x, W, b, residual=r)
    s.synchronize()
    done()
    assert torch.equal(y, want)


# ------------------------------------------------------------------ query / key norm with rotation

def qk64(x, gamma, table, positions, interleaved, eps):
    xd = x.double()
    n = xd / torch.sqrt((xd * xd).mean(-1, keepdim=True) + eps)
    if gamma is not None:
        n = n * gamma.double()
    half = table.shape[1] // 2
    cs = table[positions.long()].double()
    c, s = cs[:, None, :half], cs[:, None, half:]
    i = torch.arange(half, device=x.device)
    lo, hi = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    y, size = n.clone(), n.abs().clone()
    y[..., lo], y[..., hi] = n[..., lo] * c - n[..., hi] * s, n[..., hi] * c + n[..., lo] * s
    size[..., lo] = (n[..., lo] * c).abs() + (n[..., hi] * s).abs()
    size[..., hi] = (n[..., hi] * c).abs() + (n[..., lo] * s).abs()
    return y, size


def check_qk(y, x, gamma, table, positions, interleaved, eps=1e-6):
    ref, size = qk64(x, gamma, table, positions, interleaved, eps)
    tol = HALF_STEP * ref.abs() + (x.shape[2] / 2 + 10) * 2.0 ** -24 * size + 1e-30
    over = ((y.double() - ref).abs() - tol).max().item()
    assert over <= 0, f"beyond the tolerance by {over}"


def qk_inputs(T, Hq, Hk, D, seed, P=4096, gamma=True):
    qkv = rnd(T, Hq + 2 * Hk, D, seed=seed)
    g = torch.Generator(device=DEV)
    g.manual_seed(seed + 1)
    pos = torch.randint(0, P, (T,), generator=g, device=DEV)
    gq, gk = (1 + rnd(D, seed=seed + 2, scale=0.2), 1 + rnd(D, seed=seed + 3, scale=0.2)) if gamma else (None, None)
    return qkv[:, :Hq], qkv[:, Hq:Hq + Hk], gq, gk, pos


@pytest.mark.parametrize("T", [1, 2, 7, 64, 1021])
@pytest.mark.parametrize("Hq,Hk,D,rot,inter", [(32, 8, 128, 128, False), (32, 8, 128, 64, True), (6, 3, 80, 32, True), (6, 3, 80, 80, False),
                                               (1, 1, 8, 8, True), (3, 1, 16, 16, False), (5, 2, 24, 16, False), (4, 4, 64, 48, False),
                                               (7, 1, 96, 96, True), (2, 1, 256, 256, False), (9, 3, 192, 64, False), (1, 1, 248, 240, True)])
def test_qk_norm_rope(T, Hq, Hk, D, rot, inter):
    q, k, gq, gk, pos = qk_inputs(T, Hq, Hk, D, T + D + rot)
    table = kb.rope_table(4096, rot, device=DEV)
    yq, yk = kb.qk_norm_rope(q, k, gq, gk, table, pos, interleaved=inter)
    iq, ik = kb.qk_norm_rope(q, k, gq, None, table, pos.int(), interleaved=inter)
    done()
    check_qk(yq, q, gq, table, pos, inter)
    check_qk(yk, k, gk, table, pos, inter)
    check_qk(ik, k, None, table, pos, inter)
    assert torch.equal(iq, yq)


@pytest.mark.parametrize("T,Hq,Hk", [(16384, 32, 8), (20000, 5, 1), (3, 300, 70)])
def test_qk_norm_rope_many_rows(T, Hq, Hk):
    q, k, gq, gk, pos = qk_inputs(T, Hq, Hk, 128, 3)
    table = kb.rope_table(4096, 128, device=DEV)
    yq, yk = kb.qk_norm_rope(q, k, gq, gk, table, pos)
    done()
    check_qk(yq, q, gq, table, pos, False)
    check_qk(yk, k, gk, table, pos, False)


@pytest.mark.parametrize("seed", range(3))
def test_qk_norm_rope_random_shapes(seed):
    import random
    r = random.Random(2000 + seed)
    for i in range(30):
        inter, D = r.random() < 0.5, 8 * r.randint(2, 32)
        step = 8 if inter else 16
        rot, T = step * r.randint(1, D // step), int(math.exp(r.uniform(0, math.log(9000))))
        Hq, Hk = r.randint(1, 20), r.randint(1, 9)
        q, k, gq, gk, pos = qk_inputs(T, Hq, Hk, D, 10 * i + seed, gamma=r.random() < 0.7)
        table = kb.rope_table(4096, rot, device=DEV)
        yq, yk = kb.qk_norm_rope(q, k, gq, gk, table, pos, interleaved=inter)
        done()
        check_qk(yq, q, gq, table, pos, inter)
        check_qk(yk, k, gk, table, pos, inter)


@pytest.mark.parametrize("inter", [False, True])
def test_qk_norm_rope_in_place_and_other_layouts(inter):
    T, Hq, Hk, D = 50, 6, 2, 64
    table = kb.rope_table(4096, 64, device=DEV)
    qkv = rnd(T, Hq + 2 * Hk, D, seed=4)
    keep = qkv.clone()
    _, _, gq, gk, pos = qk_inputs(T, Hq, Hk, D, 5)
    q, k = qkv[:, :Hq], qkv[:, Hq:Hq + Hk]
    want = kb.qk_norm_rope(q, k, gq, gk, table, pos, interleaved=inter)
    kb.qk_norm_rope(q, k, gq, gk, table, pos, interleaved=inter, out=(q, k))
    done()
    check_qk(want[0], keep[:, :Hq], gq, table, pos, inter)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    assert torch.equal(qkv[:, Hq + Hk:], keep[:, Hq + Hk:])           # v is left alone
    heads_first = torch.full((Hq + 1, T + 3, D + 8), 7.0, dtype=BF16, device=DEV)   # [heads, tokens, channels] with margins
    oq = heads_first[:Hq, 1:1 + T, :D].transpose(0, 1)
    ok = torch.empty(T, Hk, D, dtype=BF16, device=DEV)
    qt = keep[:, :Hq].transpose(0, 1).contiguous().transpose(0, 1)
    kb.qk_norm_rope(qt, keep[:, Hq:Hq + Hk], gq, gk, table, pos, interleaved=inter, out=(oq, ok))
    done()
    assert torch.equal(oq, want[0]) and torch.equal(ok, want[1])
    mask = torch.ones_like(heads_first, dtype=torch.bool)
    mask[:Hq, 1:1 + T, :D] = False
    assert bool((heads_first[mask] == 7.0).all())


def test_qk_norm_rope_table_slice_zero_rows_and_non_finite_values():
    T, D = 8, 64
    q, k, gq, gk, pos = qk_inputs(T, 2, 1, D, 6)
    table = kb.rope_table(4096, 96, device=DEV)[:, :64]     # leading dimension 96: the first 32 columns cos, the next 32 "sin"
    q = q.clone()
    q[1] = 0
    q[2, 0, 5] = float("inf")
    q[3, 1, 60] = float("nan")
    yq, yk = kb.qk_norm_rope(q, k, gq, gk, table, pos)
    done()
    assert bool((yq[1] == 0).all())
    assert bool(yq[3, 1].isnan().all()) and bool(yq[3, 0].isfinite().all()) and bool(yq[2, 1].isfinite().all())
    rows = [0, 1, 4, 5, 6, 7]
    check_qk(yq[rows], q[rows], gq, table, pos[rows], False)
    check_qk(yk, k, gk, table, pos, False)


def test_qk_norm_rope_position_outside_the_table():
    q, k, gq, gk, pos = qk_inputs(6, 2, 1, 64, 7)
    table = kb.rope_table(4096, 64, device=DEV)
    good = kb.qk_norm_rope(q, k, gq, gk, table, pos)
    done()
    for bad in (4096, -1, 2 ** 40):
        pos2 = pos.clone()
        pos2[4] = bad
        out = (torch.full_like(good[0], 7.0), torch.full_like(good[1], 7.0))
        kb.qk_norm_rope(q, k, gq, gk, table, pos2, out=out)
        with pytest.raises(RuntimeError, match="position"):
            kb.check_status()
        for o, g in zip(out, good):
            assert bool((o[4] == 7.0).all())
            assert torch.equal(o[[0, 1, 2, 3, 5]], g[[0, 1, 2, 3, 5]])
    kb.check_status()


def test_qk_norm_rope_refusals_and_empty():
    q, k, gq, gk, pos = qk_inputs(6, 2, 1, 64, 8)
    table = kb.rope_table(128, 64, device=DEV)
    for args in ((q, k[:5], gq, gk, table, pos), (q, k, gq[:32], gk, table, pos), (q, k, gq, gk.float(), table, pos),
                 (q, k, gq, gk, table.double(), pos), (q, k, gq, gk, table[:, :24], pos), (q, k, gq, gk, table, pos[:5]),
                 (q, k, gq, gk, table, pos.float()), (q.float(), k, gq, gk, table, pos), (q[..., ::2], k[..., ::2], None, None, table, pos),
                 (q[0], k[0], gq, gk, table, pos)):
        with pytest.raises(ValueError):
            kb.qk_norm_rope(*args)
    with pytest.raises(ValueError, match="shares memory"):
        kb.qk_norm_rope(q, k, gq, gk, table, pos, out=(torch.empty_like(q), q[:, :1]))
    a, b = kb.qk_norm_rope(q[:0], k[:0], gq, gk, table, pos[:0])
    assert a.shape == (0, 2, 64) and b.shape == (0, 1, 64)


# ------------------------------------------------------------------ the cache

def e4m3_grid():
    v = torch.arange(256, dtype=torch.uint8).view(E4M3).double()
    return v[v.isfinite() & (v >= 0)].unique()


def quant64(x):
    """Codes (as values) and scales by the definition: the nearest e4m3 value of the exact quotient, ties to even."""
    xd = x.double().cpu()
    a = xd.abs().nan_to_num(nan=0.0, posinf=math.inf).amax(-1).clamp(min=2.0 ** -100)
    v = 448 * xd.abs() / a[..., None]          # 64 bits hold the quotient of two 8-bit numbers far past any midpoint
    grid = e4m3_grid()
    hi = torch.searchsorted(grid, v.nan_to_num(nan=0.0)).clamp(max=len(grid) - 1)
    lo = (hi - 1).clamp(min=0)
    up = grid[hi] - v < v - grid[lo]
    tie = grid[hi] - v == v - grid[lo]
    pick = torch.where(up | (tie & (hi % 2 == 0)), hi, lo)   # neighbours alternate between even and odd codes
    val = torch.where(v.isnan(), v, torch.where(v == grid[hi], grid[hi], grid[pick]))
    return torch.where(xd < 0, -val, val), (a / 448).float()


def new_cache(pages, page, H, D):
    made = []
    for _ in range(2):
        made += [torch.full((pages, page, H, D), 0x31, dtype=torch.uint8, device=DEV).view(E4M3),
                 torch.full((pages, page, H), 7.0, device=DEV)]
    return made


def check_written(cache, k, v, slots):
    pages, page, H, D = cache[0].shape
    slots = slots.cpu().long()
    for x, codes, scales in ((k, cache[0], cache[1]), (v, cache[2], cache[3])):
        want_c = torch.full((pages * page, H, D), 0x31, dtype=torch.uint8).view(E4M3).double()
        want_s = torch.full((pages * page, H), 7.0)
        val, sc = quant64(x)
        keep = slots >= 0
        want_c[slots[keep]] = val[keep]
        want_s[slots[keep]] = sc[keep]
        got = codes.cpu().to(torch.float32).double().reshape(pages * page, H, D)
        assert torch.equal(got.nan_to_num(nan=999.0), want_c.nan_to_num(nan=999.0))
        assert torch.equal(scales.cpu().reshape(pages * page, H), want_s)


@pytest.mark.parametrize("T", [1, 5, 64, 1000])
@pytest.mark.parametrize("H,D,page", [(8, 128, 16), (1, 8, 1), (5, 96, 24), (3, 80, 7), (2, 256, 64), (16, 64, 128), (1, 248, 5)])
def test_kv_cache_write(T, H, D, page):
    pages = -(-T // page) + 2
    kv = rnd(T, 3 * H, D, seed=T + H + D)
    k, v = kv[:, H:2 * H], kv[:, 2 * H:]
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(T))[:T].to(DEV)
    slots[::7] = -1
    cache = new_cache(pages, page, H, D)
    kb.kv_cache_write(k, v, slots, *cache)
    other = new_cache(pages, page, H, D)
    kb.kv_cache_write(k, v, slots.int(), *other)
    done()
    check_written(cache, k, v, slots)
    for a, b in zip(cache, other):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_kv_cache_write_every_pair_of_magnitudes():
    """Every bf16 significand against every largest value's: all quotients, exact midpoints among them, and both signs."""
    m = torch.arange(128, 256, dtype=torch.float64)
    top = m[:, None, None] / 128                                   # the row's largest value: 128 of them, in [1, 2)
    e = torch.arange(0, 20, dtype=torch.float64)
    x = (m / 256)[None, None, :] * (2.0 ** -e)[None, :, None] * torch.ones_like(top)   # below it, down to underflow
    x = torch.cat([top.expand(128, 20, 1), x, -x[..., :119]], dim=-1).to(BF16).to(DEV)  # [128, 20, 248]
    T = 128
    cache = new_cache(T, 1, 20, 248)
    slots = torch.arange(T, device=DEV)
    kb.kv_cache_write(x, -x, slots, *cache)
    done()
    check_written(cache, x, -x, slots)


def test_kv_cache_write_zeros_tiny_and_non_finite_rows():
    T, H, D = 8, 2, 64
    k, v = rnd(T, H, D, seed=1), rnd(T, H, D, seed=2)
    k[0] = 0
    k[1] *= 2.0 ** -110                      # below the floor of the scale
    k[2] = torch.tensor(1e-40).to(BF16)      # subnormal
    k[3] = 3e38
    k[4, 0, 3] = float("nan")
    k[5] = float("nan")
    v[6, 1, 9] = float("inf")
    v[7, 0, 2] = float("-inf")
    cache = new_cache(2, 4, H, D)
    slots = torch.arange(T, device=DEV)
    kb.kv_cache_write(k, v, slots, *cache)
    done()
    check_written(cache, k, v, slots)
    ko, vo = kb.kv_cache_read(*cache, torch.tensor([[0, 1]], dtype=torch.int32, device=DEV), torch.tensor([0, 8], dtype=torch.int32, device=DEV), 8)
    done()
    assert bool((ko[0] == 0).all()) and bool(ko[:4].isfinite().all())
    assert ko[4, 0].isnan().nonzero().tolist() == [[3]] and bool(ko[5].isnan().all())
    assert bool(vo[6, 1].isnan().all()) and bool(vo[6, 0].isfinite().all()) and bool(vo[7, 0].isnan().all())


def test_kv_cache_write_slot_outside_the_cache():
    T, H, D = 6, 2, 64
    k, v = rnd(T, H, D, seed=3), rnd(T, H, D, seed=4)
    for bad in (8, 2 ** 33, 2 ** 62):
        cache = new_cache(2, 4, H, D)
        slots = torch.tensor([0, 1, bad, 3, -5, 7], device=DEV)
        kb.kv_cache_write(k, v, slots, *cache)
        with pytest.raises(RuntimeError, match=f"slot {bad}"):
            kb.check_status()
        slots[2] = -1
        check_written(cache, k, v, slots)
    kb.check_status()


@pytest.mark.parametrize("layout", ["pages in turn", "side by side", "heads outside"])
def test_kv_cache_layouts(layout):
    pages, page, H, D, T = 5, 8, 3, 64, 33
    if layout == "pages in turn":
        codes = torch.zeros(pages, 2, page, H, D, dtype=torch.uint8, device=DEV).view(E4M3)
        scales = torch.zeros(pages, 2, page, H, device=DEV)
        cache = [codes[:, 0], scales[:, 0], codes[:, 1], scales[:, 1]]
    elif layout == "side by side":
        codes = torch.zeros(pages, page, H, 2, D + 8, dtype=torch.uint8, device=DEV).view(E4M3)
        scales = torch.zeros(pages, page, H, 2, device=DEV)
        cache = [codes[..., 0, :D], scales[..., 0], codes[..., 1, :D], scales[..., 1]]
    else:
        codes = torch.zeros(2, H, pages, page, D, dtype=torch.uint8, device=DEV).view(E4M3)
        scales = torch.zeros(2, H, pages, page, device=DEV)
        cache = [t for i in range(2) for t in (codes[i].permute(1, 2, 0, 3), scales[i].permute(1, 2, 0))]
    plain = [t.contiguous() for t in cache]
    k, v = rnd(T, H, D, seed=5), rnd(T, H, D, seed=6)
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(1))[:T].to(DEV)
    kb.kv_cache_write(k, v, slots, *cache)
    kb.kv_cache_write(k, v, slots, *plain)
    table = torch.tensor([[3, 0, 4], [1, 2, -1]], dtype=torch.int32, device=DEV)
    cu = torch.tensor([0, 20, 33], dtype=torch.int32, device=DEV)
    a, b = kb.kv_cache_read(*cache, table, cu, 33), kb.kv_cache_read(*plain, table, cu, 33)
    done()
    for x, y in zip(cache, plain):
        assert torch.equal(x.contiguous().view(torch.uint8), y.view(torch.uint8))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def random_cache(pages, page, H, D, seed):
    g = torch.Generator().manual_seed(seed)
    made = []
    for _ in range(2):
        codes = torch.randint(0, 256, (pages, page, H, D), generator=g, dtype=torch.uint8)
        codes[(codes & 0x7f) == 0x7f] = 0x40
        made += [codes.to(DEV).view(E4M3), torch.exp(torch.randn(pages, page, H, generator=g) * 3).to(DEV)]
    return made


def read_ref(cache, table, lens, page):
    """On the CPU, token by token; the product in fp32 and its rounding to bf16 are both IEEE."""
    out = []
    for codes, scales in (cache[:2], cache[2:]):
        c, s = codes.cpu().to(torch.float32), scales.cpu()
        rows = [c[table[b][i // page], i % page] * s[table[b][i // page], i % page][:, None] for b, n in enumerate(lens) for i in range(n)]
        out.append(torch.stack(rows).to(BF16) if rows else torch.zeros(0, *codes.shape[2:], dtype=BF16))
    return out


@pytest.mark.parametrize("lens", [[1], [0, 1], [0, 0, 5, 0], [17, 0, 1, 16, 33], [3] * 40, [1, 0] * 600, [700, 2, 90]])
@pytest.mark.parametrize("H,D,page", [(8, 128, 16), (1, 8, 1), (5, 96, 24), (2, 256, 7), (3, 72, 64)])
def test_kv_cache_read(lens, H, D, page):
    used = [-(-n // page) for n in lens]
    pages = sum(used) + 2
    cache = random_cache(pages, page, H, D, 11)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(2)).tolist()
    width = max(max(used), 1) + 1
    table, at = [], 0
    for u in used:
        table.append(order[at:at + u] + [-1] * (width - u))
        at += u
    ends = [0]
    for n in lens:
        ends.append(ends[-1] + n)
    total = ends[-1] + 3
    dt, cu = torch.tensor(table, dtype=torch.int32, device=DEV), torch.tensor(ends, dtype=torch.int32, device=DEV)
    want = read_ref(cache, table, lens, page)
    fresh = kb.kv_cache_read(*cache, dt, cu, total)
    both = torch.full((total + 2, H, 2 * D + 8), 7.0, dtype=BF16, device=DEV)
    out = (both[1:1 + total, :, :D], both[1:1 + total, :, D + 8:])
    kb.kv_cache_read(*cache, dt, cu, total, out=out)
    short = kb.kv_cache_read(*cache, dt, cu, max(total - 4, 1))
    done()
    n = ends[-1]
    for f, o, s, w in zip(fresh, out, short, want):
        assert torch.equal(f[:n].cpu(), w) and bool((f[n:] == 0).all())
        assert torch.equal(o[:n].cpu(), w) and bool((o[n:] == 7.0).all())      # rows behind the last sequence: as they were
        assert torch.equal(s[:total - 4].cpu(), w[:total - 4])
    assert bool((both[0] == 7.0).all()) and bool((both[-1] == 7.0).all()) and bool((both[:, :, D:D + 8] == 7.0).all())


def test_kv_cache_read_bad_pages_and_short_tables():
    page, H, D = 4, 2, 64
    cache = random_cache(3, page, H, D, 12)
    cu = torch.tensor([0, 6, 9], dtype=torch.int32, device=DEV)
    good = kb.kv_cache_read(*cache, torch.tensor([[0, 1], [2, -1]], dtype=torch.int32, device=DEV), cu, 9)
    done()
    for bad in (3, -1, 2 ** 30, -2 ** 31):
        out = (torch.full_like(good[0], 7.0), torch.full_like(good[1], 7.0))
        kb.kv_cache_read(*cache, torch.tensor([[0, bad], [2, -1]], dtype=torch.int32, device=DEV), cu, 9, out=out)
        with pytest.raises(RuntimeError, match=f"page {bad}"):
            kb.check_status()
        for o, g in zip(out, good):
            assert torch.equal(o[:4], g[:4]) and bool((o[4:6] == 7.0).all()) and torch.equal(o[6:], g[6:])
    for cut in ([[0], [2]], [[], []]):            # sequences longer than their rows of the table
        fresh = kb.kv_cache_read(*cache, torch.tensor(cut, dtype=torch.int32, device=DEV).view(2, -1), cu, 9)
        with pytest.raises(RuntimeError, match="page"):
            kb.check_status()
        for o, g in zip(fresh, good):             # a fresh output holds zeros there
            n = 4 if cut[0] else 0
            assert torch.equal(o[:n], g[:n]) and bool((o[n:6] == 0).all())
    for ends in ([5, 6, 9], [0, 9, 4], [-3, 2, 2 ** 31 - 1]):     # lengths that make no sense stay inside the table
        kb.kv_cache_read(*cache, torch.tensor([[0, 1], [2, -1]], dtype=torch.int32, device=DEV),
                         torch.tensor(ends, dtype=torch.int32, device=DEV), 9)
        torch.cuda.synchronize()
        try:
            kb.check_status()
        except RuntimeError:
            pass
    none = kb.kv_cache_read(*cache, torch.zeros(0, 2, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV), 2)
    done()
    assert bool((none[0] == 0).all()) and bool((none[1] == 0).all())
    assert kb.kv_cache_read(*cache, torch.zeros(0, 2, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV), 0)[0].shape == (0, H, D)


def test_kv_cache_beyond_32_bit_offsets():
    """Pages that lie more than 2^32 bytes into the cache, and scales more than 2^32 bytes into theirs."""
    H, D, page = 2, 64, 4
    gap = 1 << 31
    codes = torch.empty(2 * gap + 2 * page * H * D, dtype=torch.uint8, device=DEV)
    scales = torch.empty((1 << 30) + 2 * page * H + (1 << 29), dtype=torch.float32, device=DEV)
    cache = []
    for i in range(2):
        cache += [codes[i * page * H * D:].as_strided((3, page, H, D), (gap, H * D, D, 1)).view(E4M3),
                  scales[i * page * H:].as_strided((3, page, H), (1 << 29, H, 1))]
    k, v = rnd(12, H, D, seed=7), rnd(12, H, D, seed=8)
    slots = torch.arange(12, device=DEV)
    kb.kv_cache_write(k, v, slots, *cache)
    ko, vo = kb.kv_cache_read(*cache, torch.tensor([[0, 1, 2]], dtype=torch.int32, device=DEV),
                              torch.tensor([0, 12], dtype=torch.int32, device=DEV), 12)
    done()
    for x, y in ((k, ko), (v, vo)):
        val, sc = quant64(x)
        assert torch.equal(y.cpu(), (val.float() * sc[..., None]).to(BF16))


def test_kv_cache_refusals():
    cache = new_cache(2, 4, 2, 64)
    k, v = rnd(4, 2, 64, seed=1), rnd(4, 2, 64, seed=2)
    slots = torch.arange(4, device=DEV)
    c0, s0, c1, s1 = cache
    for args in ((k, v[:3], slots, *cache), (k[:, :1], v[:, :1], slots, *cache), (k.half(), v.half(), slots, *cache), (k, v, slots[:3], *cache),
                 (k, v, slots.float(), *cache), (k, v, slots, c0.view(torch.uint8), s0, c1, s1), (k, v, slots, c0, s0[:1], c1, s1),
                 (k, v, slots, c0, s0, c1[:1], s1), (k, v, slots, c0, s0.double(), c1, s1)):
        with pytest.raises(ValueError):
            kb.kv_cache_write(*args)
    with pytest.raises(ValueError, match="shares memory"):
        kb.kv_cache_write(k, v, slots, c0, s0, c0, s1)
    kb.kv_cache_write(k[:0], v[:0], slots[:0], *cache)
    table, cu = torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.tensor([0, 4], dtype=torch.int32, device=DEV)
    for args, kw in (((table.long(), cu, 4), {}), ((table, cu.long(), 4), {}), ((table, cu[:1], 4), {}), ((table, cu, -1), {}),
                     ((table, cu, 4), dict(out=(k, v[:3]))), ((table, cu, 4), dict(out=(k, k)))):
        with pytest.raises(ValueError):
            kb.kv_cache_read(*cache, *args, **kw)
    done()


# ------------------------------------------------------------------ together

def layer(h, w, cache, slots, table, cu, positions, rope, Hq, Hk, D, lens):
    """One decoder layer around an attention of the caller's own: what the operators are for."""
    T = h.shape[0]
    qkv = kb.rmsnorm_linear(h, w["g1"], w["qkv"]).view(T, Hq + 2 * Hk, D)
    q, k = kb.qk_norm_rope(qkv[:, :Hq], qkv[:, Hq:Hq + Hk], w["gq"], w["gk"], rope, positions)
    kb.kv_cache_write(k, qkv[:, Hq + Hk:], slots, *cache)
    ks, vs = kb.kv_cache_read(*cache, table, cu, sum(lens))
    outs, at = [], 0
    for b, n in enumerate(lens):       # one new token per sequence, over all of it
        kk, vv = (t[at:at + n].float().repeat_interleave(Hq // Hk, dim=1) for t in (ks, vs))
        p = torch.softmax(torch.einsum("hd,nhd->hn", q[b].float(), kk) / math.sqrt(D), dim=-1)
        outs.append(torch.einsum("hn,nhd->hd", p, vv))
        at += n
    att = torch.stack(outs).to(BF16).view(T, Hq * D)
    h = kb.linear(att, w["o"], residual=h)
    return kb.linear(kb.rmsnorm_swiglu(h, w["g2"], w["gu"]), w["down"], residual=h)


def layer64(h, w, hist, rope, positions, Hq, Hk, D, lens):
    h = h.double()

    def norm(x, g):
        return x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * g.double()

    T = h.shape[0]
    qkv = (norm(h, w["g1"]) @ w["qkv"].double().t()).view(T, Hq + 2 * Hk, D)
    q, _ = qk64(qkv[:, :Hq], w["gq"], rope, positions, False, 1e-6)
    k, _ = qk64(qkv[:, Hq:Hq + Hk], w["gk"], rope, positions, False, 1e-6)
    outs = []
    for b, n in enumerate(lens):
        kk = torch.cat([hist[b][0].double(), k[b:b + 1]]).repeat_interleave(Hq // Hk, dim=1)
        vv = torch.cat([hist[b][1].double(), qkv[b:b + 1, Hq + Hk:]]).repeat_interleave(Hq // Hk, dim=1)
        p = torch.softmax(torch.einsum("hd,nhd->hn", q[b], kk) / math.sqrt(D), dim=-1)
        outs.append(torch.einsum("hn,nhd->hd", p, vv))
    h = h + torch.stack(outs).view(T, Hq * D) @ w["o"].double().t()
    gu = norm(h, w["g2"]) @ w["gu"].double().t()
    g, u = gu.chunk(2, dim=-1)
    return h + (g * torch.sigmoid(g) * u) @ w["down"].double().t()


@pytest.mark.parametrize("graph", [False, True])
def test_decode_step_through_a_layer(graph):
    """Prompt tokens written, then one token per sequence through a layer, eager and as a captured graph, against 64 bits.

    Each operator's own tolerance is tested above; here the e4m3 cache dominates: half a step of 2^-4 relative to a value on
    every key and value read, averaged over the sequence.  Keys move the scores (sqrt(D) spread) by at most 2^-4 of a unit,
    values the output by 2^-4 of their size: with both, an output of the attention is off by less than an eighth of the
    values' norm, and it adds to a residual stream of the same size."""
    Hq, Hk, D, dim, ff, page = 8, 2, 64, 512, 1024, 16
    lens = [1, 17, 40, 128]
    T = len(lens)
    w = {"g1": 1 + rnd(dim, seed=1, scale=0.1), "g2": 1 + rnd(dim, seed=2, scale=0.1), "gq": 1 + rnd(D, seed=3, scale=0.1),
         "gk": 1 + rnd(D, seed=4, scale=0.1), "qkv": rnd((Hq + 2 * Hk) * D, dim, seed=5, scale=dim ** -0.5),
         "o": rnd(dim, Hq * D, seed=6, scale=(Hq * D) ** -0.5), "gu": rnd(2 * ff, dim, seed=7, scale=dim ** -0.5),
         "down": rnd(dim, ff, seed=8, scale=ff ** -0.5)}
    rope = kb.rope_table(256, D, device=DEV)
    used = [-(-n // page) for n in lens]
    table = torch.full((T, max(used)), -1, dtype=torch.int32)
    order, at = torch.randperm(sum(used), generator=torch.Generator().manual_seed(3)).int(), 0
    for b, u in enumerate(used):
        table[b, :u] = order[at:at + u]
        at += u
    cache = [torch.zeros(sum(used), page, Hk, D, dtype=torch.uint8, device=DEV).view(E4M3) if i % 2 == 0 else
             torch.zeros(sum(used), page, Hk, device=DEV) for i in range(4)]
    hist = []
    for b, n in enumerate(lens):
        k, v = rnd(n - 1, Hk, D, seed=20 + b), rnd(n - 1, Hk, D, seed=30 + b)
        hist.append((k, v))
        i = torch.arange(n - 1)
        kb.kv_cache_write(k, v, (table[b, i // page].long() * page + i % page).to(DEV), *cache)
    last = torch.tensor(lens) - 1
    slots = (table[torch.arange(T), last // page].long() * page + last % page).to(DEV)
    ends = torch.tensor([0] + lens).cumsum(0).int().to(DEV)
    h = rnd(T, dim, seed=40)
    args = (h, w, cache, slots, table.to(DEV), ends, last.to(DEV), rope, Hq, Hk, D, lens)
    if graph:
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            layer(*args)
            s.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                y = layer(*args)
        h.copy_(rnd(T, dim, seed=41))     # the replay sees new inputs
        g.replay()
    else:
        y = layer(*args)
    done()
    ref = layer64(h, w, hist, rope, last.to(DEV), Hq, Hk, D, lens)
    err = (y.double() - ref).norm(dim=-1) / ref.norm(dim=-1)
    assert bool((err <= 0.125).all()), err
    # the prompts' rows are still what was written
    ko, vo = kb.kv_cache_read(*cache, table.to(DEV), ends, sum(lens))
    done()
    at = 0
    for (k, v), n in zip(hist, lens):
        for x, got in ((k, ko), (v, vo)):
            val, sc = quant64(x)
            assert torch.equal(got[at:at + n - 1].cpu(), (val.float() * sc[..., None]).to(BF16))
        at += n


def test_operators_in_a_graph_report_bad_indices():
    q, k, gq, gk, pos = qk_inputs(4, 2, 1, 64, 90)
    table = kb.rope_table(4096, 64, device=DEV)
    out = (torch.zeros(4, 2, 64, dtype=BF16, device=DEV), torch.zeros(4, 1, 64, dtype=BF16, device=DEV))
    kb.qk_norm_rope(q, k, gq, gk, table, pos, out=out)
    done()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        kb.qk_norm_rope(q, k, gq, gk, table, pos, out=out)
    g.replay()
    done()
    pos[2] = 4096
    g.replay()
    with pytest.raises(RuntimeError, match="position 4096, row 2"):
        kb.check_status()
    pos[2] = 5
    g.replay()
    done()
    check_qk(out[0], q, gq, table, pos, False)


def test_chains_without_synchronising():
    """Each operator launched right behind the one that writes its inputs."""
    Hq, Hk, D, dim, T = 8, 2, 128, 1024, 16
    x, W = rnd(T, dim, seed=1), rnd((Hq + 2 * Hk) * D, dim, seed=2, scale=dim ** -0.5)
    Wo = rnd(dim, Hq * D, seed=3, scale=0.03)
    table, pos = kb.rope_table(64, D, device=DEV), torch.arange(T, device=DEV)
    pt, cu = torch.tensor([[0]], dtype=torch.int32, device=DEV), torch.tensor([0, T], dtype=torch.int32, device=DEV)

    def run(sync):
        cache = new_cache(1, T, Hk, D)
        got = []
        for op in range(5):
            if op == 0:
                qkv = kb.linear(x, W).view(T, -1, D)
            elif op == 1:
                q, k = kb.qk_norm_rope(qkv[:, :Hq], qkv[:, Hq:Hq + Hk], None, None, table, pos)
            elif op == 2:
                kb.kv_cache_write(k, qkv[:, Hq + Hk:], pos, *cache)
            elif op == 3:
                got += kb.kv_cache_read(*cache, pt, cu, T)
            else:
                got.append(kb.linear(q.view(T, -1), Wo, residual=x))
            if sync:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        return got

    want = run(True)
    for _ in range(50):
        for a, b in zip(run(False), want):
            assert torch.equal(a, b)
    done()
