"""token_embedding: rows against the fp32 product rounded once more to the type,
gradients against float64.

A gradient is a sum of n fp32 terms, in whatever grouping: within n e of the sum of
absolute terms (e = 2^-24), then scaled (1 e) and rounded to the type.
"""

from __future__ import annotations

import math

import pytest
import torch

import myelin_amd as myelin
from myelin_amd import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}


def _case(**kw):
    print("case:", " ".join(f"{k}={v}" for k, v in kw.items()), flush=True)


def _half(dt):
    return torch.finfo(dt).eps / 2


def _want(tokens, weight, scale, padding):
    rows = (weight.detach().float() * torch.tensor(scale, dtype=torch.float32, device=weight.device)).to(weight.dtype)
    V = weight.shape[0]
    inside = (tokens >= 0) & (tokens < V)
    y = torch.where(inside[..., None], rows[tokens.clamp(0, V - 1)], math.nan)
    return y if padding is None else torch.where((tokens == padding)[..., None], 0.0, y)


def _check_grad(got, tokens, g, V, scale, padding):
    flat, g = tokens.reshape(-1).cpu(), g.detach().double().cpu().reshape(tokens.numel(), -1)
    real = (flat >= 0) & (flat < V)
    if padding is not None:
        real &= flat != padding
    flat, g = flat[real], g[real]
    total = torch.zeros(V, g.shape[1], dtype=torch.float64).index_add_(0, flat, g)
    size = torch.zeros_like(total).index_add_(0, flat, g.abs())
    count = torch.bincount(flat, minlength=V)[:, None]
    s32 = float(torch.tensor(scale, dtype=torch.float32))
    want, room = total * s32, (count + 2) * 2.0**-24 * size * abs(s32)
    room = room + _half(got.dtype) * (want.abs() + room) + 1e-38
    assert bool(((got.double().cpu() - want).abs() <= room).all())
    assert bool((got.cpu()[count[:, 0] == 0] == 0).all())


def _grad(tokens, weight, g, **kw):
    w = weight.detach().clone().requires_grad_()
    y = myelin.token_embedding(tokens, w, **kw)
    (gw,) = torch.autograd.grad(y, w, g)
    assert gw.shape == w.shape and gw.dtype == w.dtype
    return gw


SIZES = [((1,), 1, 1), ((), 5, 3), ((3,), 7, 64), ((7, 5), 11, 130), ((64, 32), 50, 128), ((1000,), 3, 33),
         ((4097,), 1000, 17), ((300, 7), 2, 8), ((129,), 100003, 5), ((20000,), 700, 24), ((33, 1000), 40000, 9),
         ((70000,), 5, 4), ((17000,), 300000, 3), ((2,), 3, 5000), ((140000,), 513, 2), ((40000,), 30000, 2),
         ((270000,), 200, 3), ((280000,), 90000, 2), ((265000,), 40, 5)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,V,D", SIZES)
def test_rows_and_gradients(shape, V, D, dtype):
    _case(test="embedding", shape=shape, V=V, D=D, dtype=dtype)
    g = torch.Generator().manual_seed(V + D)
    weight = torch.randn(V, D, generator=g).to(DTYPES[dtype]).to(DEV)
    uniform = torch.randint(0, V, shape, generator=g)
    # frequencies that fall as 1 / rank
    skewed = (torch.exp(torch.rand(shape, generator=g, dtype=torch.float64) * math.log(V + 1)).long() - 1).clamp(0, V - 1)
    for tokens, scale, padding in ((uniform, 1.0, None), (skewed, D**0.5, None), (skewed, -0.3, 0), (uniform, 3.0, -100)):
        tokens = tokens.to(DEV)
        y = myelin.token_embedding(tokens, weight, scale=scale, padding_index=padding)
        assert y.dtype == weight.dtype and torch.equal(y, _want(tokens, weight, scale, padding))
        gy = torch.randn(*shape, D, generator=g).to(DTYPES[dtype]).to(DEV)
        gw = _grad(tokens, weight, gy, scale=scale, padding_index=padding)
        _check_grad(gw, tokens, gy, V, scale, padding)
        # int32 tokens, and the same bits again
        same = _grad(tokens.int(), weight, gy, scale=scale, padding_index=padding)
        assert torch.equal(gw, same)


@pytest.mark.parametrize("M", [1, 63, 64, 65, 128, 1000, 4096, 5000, 16384, 16385, 40000, 300000])
def test_one_token_and_all_of_them(M):
    """A run of every position, alone and between others."""

    for dtype in DTYPES:
        _case(test="embedding_runs", M=M, dtype=dtype)
        g = torch.Generator().manual_seed(M)
        weight = torch.randn(9, 6, generator=g).to(DTYPES[dtype]).to(DEV)
        gy = torch.randn(M, 6, generator=g).to(DTYPES[dtype]).to(DEV)
        for tokens in (torch.full((M,), 4), torch.full((M,), 8), torch.full((M,), 0), torch.arange(M) % 2 * 8,
                       torch.where(torch.arange(M) < M // 3, 7, 2), torch.arange(M).clamp(max=8)):
            tokens = tokens.to(DEV)
            _check_grad(_grad(tokens, weight, gy), tokens, gy, 9, 1.0, None)


def test_the_order_of_the_positions_is_kept():
    """1, 2^24 and -2^24 in an order that shows in the sum: equal tokens' rows are
    added in order of their positions wherever they stand."""

    big = 2.0**24
    values = torch.tensor([big, 1.0, -big, 1.0])  # in order: 1; sorted otherwise: 0 or 2
    for gap in (0, 3, 200, 6000):
        M = 4 + 4 * gap
        tokens = torch.ones(M, dtype=torch.int64)
        gy = torch.zeros(M, 1)
        for i in range(4):
            tokens[i * (gap + 1)], gy[i * (gap + 1), 0] = 5, values[i]
        gw = _grad(tokens.to(DEV), torch.zeros(7, 1, device=DEV), gy.to(DEV))
        assert float(gw[5, 0]) == 1.0


@pytest.mark.parametrize("dtype", DTYPES)
def test_tokens_outside_the_table(dtype):
    _case(test="embedding_outside", dtype=dtype)
    weight = torch.randn(10, 12, device=DEV).to(DTYPES[dtype])
    tokens = torch.tensor([0, -1, 9, 10, 2**31 + 3, -(2**40), 2**62, 9, -(2**63), -100], device=DEV)
    y = myelin.token_embedding(tokens, weight, scale=2.0, padding_index=-100)
    inside = torch.tensor([0, 2, 7], device=DEV)
    assert torch.equal(y[inside], _want(tokens[inside], weight, 2.0, None))
    assert bool(y[torch.tensor([1, 3, 4, 5, 6, 8])].isnan().all()) and bool((y[9] == 0).all())
    gy = torch.full_like(y, math.nan)
    gy[inside] = 1.0
    gw = _grad(tokens, weight, gy, scale=2.0, padding_index=-100)
    assert bool((gw[0] == 2).all()) and bool((gw[9] == 4).all()) and bool((gw[1:9] == 0).all())
    # the padding row of a table: not even its NaN
    weight[3] = math.nan
    tokens = torch.tensor([3, 4, 3], device=DEV)
    y = myelin.token_embedding(tokens, weight, padding_index=3)
    assert bool((y[0] == 0).all()) and bool((y[2] == 0).all()) and torch.equal(y[1], weight[4])


def test_infinities_and_nans_stay_in_their_rows():
    for M in (50, 3000, 20000):
        tokens = torch.arange(M, device=DEV) % 37
        gy = torch.randn(M, 20, device=DEV)
        clean = _grad(tokens, torch.zeros(40, 20, device=DEV), gy)
        gy[7, 3], gy[8, 4] = math.inf, math.nan
        bad = _grad(tokens, torch.zeros(40, 20, device=DEV), gy)
        assert float(bad[7, 3]) == math.inf and bool(bad[8, 4].isnan())
        bad[7, 3], bad[8, 4] = clean[7, 3], clean[8, 4]
        assert torch.equal(bad, clean)


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts(dtype):
    g = torch.Generator().manual_seed(2)
    base = torch.randn(40, 70, generator=g).to(DTYPES[dtype]).to(DEV)
    tokens = torch.randint(0, 40, (6, 31), generator=g).to(DEV)
    for w in (base[:, :64], base[:, 1:65], base[::2, 3:], base.t(), base[:1].expand(40, 70), base[:, ::2]):
        t = tokens % w.shape[0]
        assert torch.equal(myelin.token_embedding(t, w, scale=1.5), _want(t, w, 1.5, None))
        leaf = w.detach().requires_grad_()
        gy = torch.randn(6, 31, w.shape[1], generator=g).to(w.dtype).to(DEV)
        (gw,) = torch.autograd.grad(myelin.token_embedding(t, leaf, scale=1.5), leaf, gy)
        _check_grad(gw.contiguous(), t, gy, w.shape[0], 1.5, None)
    w = base.clone().requires_grad_()
    swapped = tokens.t()
    y = myelin.token_embedding(swapped, w)
    assert torch.equal(y.detach(), _want(swapped, w, 1.0, None))
    (a,) = torch.autograd.grad(y.sum(), w)  # an expanded gradient
    count = torch.bincount(tokens.reshape(-1), minlength=40)
    assert torch.equal(a.float(), count[:, None].float().expand(40, 70).to(a.dtype).float())
    gy = torch.randn(6, 31, 70, generator=g).to(w.dtype).to(DEV).transpose(0, 1)  # not contiguous
    (a,) = torch.autograd.grad(myelin.token_embedding(swapped, w), w, gy)
    (b,) = torch.autograd.grad(myelin.token_embedding(swapped, w), w, gy.contiguous())
    assert torch.equal(a, b)


def test_no_tokens():
    w = torch.randn(5, 4, device=DEV, requires_grad=True)
    tokens = torch.empty(3, 0, dtype=torch.int64, device=DEV)
    y = myelin.token_embedding(tokens, w)
    assert y.shape == (3, 0, 4)
    (gw,) = torch.autograd.grad(y, w, torch.empty_like(y))
    assert torch.equal(gw, torch.zeros_like(w))
    # and more rows than a launch of sum_few would have workgroups
    many = torch.ones(2**23 + 100, 1, device=DEV, requires_grad=True)
    y = myelin.token_embedding(tokens, many)
    (gm,) = torch.autograd.grad(y, many, torch.empty_like(y))
    assert not bool(gm.any())
    # nothing but padding
    tokens = torch.full((100,), 2, device=DEV)
    y = myelin.token_embedding(tokens, w, padding_index=2)
    (gw,) = torch.autograd.grad(y, w, torch.ones_like(y))
    assert torch.equal(gw, torch.zeros_like(w)) and not bool(y.any())


def test_gradients_are_differences():
    """y is linear: a difference of two outputs is the product with the gradient."""

    g = torch.Generator().manual_seed(9)
    tokens = torch.randint(0, 30, (500,), generator=g).to(DEV)
    w, d = (torch.randint(-8, 9, (30, 16), generator=g).float().to(DEV) for _ in range(2))
    gy = torch.randint(-4, 5, (500, 16), generator=g).float().to(DEV)
    gw = _grad(tokens, w, gy, scale=2.0)
    up, down = (myelin.token_embedding(tokens, v, scale=2.0).double() for v in (w + d, w - d))
    # whole numbers below 2^24: exact on both sides
    assert float(((up - down) / 2 * gy.double()).sum()) == float((gw.double() * d.double()).sum())


def test_offsets_past_32_bits():
    _case(test="embedding_large")
    V, D = 2**20 + 5, 2100
    w = torch.ones(V, D, dtype=torch.bfloat16, device=DEV)
    w[-1] = 3.0
    w.requires_grad_()
    tokens = torch.tensor([V - 1, 0, V - 1, 1023], device=DEV)
    y = myelin.token_embedding(tokens, w, scale=0.5)
    assert torch.equal(y[:, 0].float(), torch.tensor([1.5, 0.5, 1.5, 0.5], device=DEV))
    (gw,) = torch.autograd.grad(y, w, torch.ones_like(y))
    assert bool((gw[-1] == 1).all()) and bool((gw[0] == 0.5).all()) and bool((gw[1023] == 0.5).all())
    assert not bool(gw[-2].any()) and int((gw[:, 0] != 0).sum()) == 3
    del w, y, gw
    M, D = 1030000, 2100
    tokens = torch.arange(M, device=DEV) % 3
    y = myelin.token_embedding(tokens, torch.tensor([[1.0], [2.0], [4.0]], dtype=torch.bfloat16,
                                                    device=DEV).repeat(1, D).requires_grad_())
    assert torch.equal(y[-4:, -1].float(), torch.tensor([1.0, 2.0, 4.0], device=DEV)[(tokens[-4:])])


def test_refusals():
    w = torch.zeros(4, 5, device=DEV)
    t = torch.zeros(3, dtype=torch.int64, device=DEV)
    f = myelin.token_embedding
    for bad, message in ((lambda: f(t, w[0]), "weight must be"), (lambda: f(t, w[:0]), "weight must be"),
                         (lambda: f(t, w[:, :0]), "weight must be"), (lambda: f(t, w.half()), "float32 or bfloat16"),
                         (lambda: f(t.cpu(), w), "same device"), (lambda: f(t.float(), w), "int64 or int32"),
                         (lambda: f(t, w, scale=math.inf), "scale must be"),
                         (lambda: f(t, w, scale=math.nan), "scale must be"), (lambda: f(t, w, scale=1e39), "scale must"),
                         (lambda: f(t, w, padding_index=2**63), "padding_index")):
        with pytest.raises(ValueError, match=message):
            bad()


def test_module():
    torch.manual_seed(3)
    m = myelin.TokenEmbedding(20, 8, scale=2.0, padding_index=0).to(DEV)
    torch.manual_seed(3)
    assert torch.equal(m.weight.detach().cpu(), torch.nn.Embedding(20, 8).weight.detach())
    t = torch.tensor([[0, 5], [7, 5]], device=DEV)
    y = m(t)
    assert torch.equal(y.detach(), _want(t, m.weight, 2.0, 0))
    y.sum().backward()
    assert torch.equal(m.weight.grad[5], torch.full((8,), 4.0, device=DEV)) and not bool(m.weight.grad[0].any())


@pytest.mark.parametrize("V", [40, 300, 40000, 70000])
@pytest.mark.parametrize("M", [4097, 131072, 131073, 524289, 1500000])
def test_positions_of_many_workgroups(M, V):
    """Sorts by digits of 6, 8 and 9 bits, by up to 128 workgroups, by more and in
    several turns of each.  Whole numbers: their sums are exact, in any order."""

    _case(test="embedding_many", M=M, V=V)
    g = torch.Generator().manual_seed(M + V)
    spread = torch.rand(M, generator=g)
    tokens = (V * spread**3).long().clamp(max=V - 1)  # small ones more often
    tokens[torch.randint(0, M, (M // 50,), generator=g)] = 2  # padding
    tokens[torch.randint(0, M, (9,), generator=g)] = V  # outside
    gy = torch.randint(-3, 4, (M, 2), generator=g).float()
    want = torch.zeros(V, 2, dtype=torch.float64)
    counted = (tokens < V) & (tokens != 2)
    want.index_add_(0, tokens[counted], gy[counted].double())
    assert float(torch.bincount(tokens).max()) * 3 < 2**24
    gw = _grad(tokens.to(DEV), torch.zeros(V, 2, device=DEV), gy.to(DEV), padding_index=2)
    assert torch.equal(gw.cpu().double(), want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,V,D", [(1, 5000, 3), (33, 2049, 64), (60, 5407, 26), (511, 4102, 73), (700, 9000, 640),
                                   (1023, 2200, 1001), (2048, 40000, 16), (2049, 40000, 16), (3000, 2500, 130)])
def test_few_positions_of_a_large_table(M, V, D, dtype):
    """A workgroup to a position, beside the sort of a few more: whole numbers, whose
    sums are exact and round once."""

    _case(test="embedding_positions", M=M, V=V, D=D, dtype=dtype)
    g = torch.Generator().manual_seed(M + V + D)
    for tokens in (torch.randint(0, V, (M,), generator=g), torch.randint(0, 9, (M,), generator=g) * (V // 9),
                   torch.full((M,), V - 1), torch.arange(M).flip(0) % V):
        tokens = tokens.clone()
        tokens[M // 2] = 3  # padding
        tokens[M // 3] = -1
        gy = torch.randint(-2, 3, (M, D), generator=g).to(DTYPES[dtype])
        want = torch.zeros(V, D, dtype=torch.float64)
        counted = (tokens >= 0) & (tokens != 3)
        want.index_add_(0, tokens[counted], gy[counted].double())
        gw = _grad(tokens.to(DEV), torch.zeros(V, D, dtype=DTYPES[dtype], device=DEV), gy.to(DEV), padding_index=3)
        assert torch.equal(gw.cpu(), want.to(DTYPES[dtype]))


@pytest.mark.parametrize("V,width", [(5000, 1), (5000, 8), (300, 300)])
def test_the_order_is_kept_in_larger_tables(V, width):
    big = 2.0**24
    values = torch.tensor([big, 1.0, -big, 1.0])
    for gap in (0, 3, 200, 500, 3000, 40000):
        M = 4 + 4 * gap
        tokens = torch.arange(M) % (V - 10) + 6
        gy = torch.zeros(M, width)
        for i in range(4):
            tokens[i * (gap + 1)], gy[i * (gap + 1)] = 5, values[i]
        gw = _grad(tokens.to(DEV), torch.zeros(V, width, device=DEV), gy.to(DEV))
        assert bool((gw[5] == 1.0).all()), gap


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,V,D", [(70, 30, 9), (300, 50, 17), (2500, 3001, 33), (5000, 1000, 301), (9, 7, 8)])
def test_rows_that_start_anywhere(M, V, D, dtype):
    """Tables and gradients that start one element behind 16 bytes, rows of odd widths
    and strides: what is beside them is neither read into results nor written."""

    _case(test="embedding_anywhere", M=M, V=V, D=D, dtype=dtype)
    g = torch.Generator().manual_seed(M + V + D)
    dt = DTYPES[dtype]
    base = torch.full((V * (D + 2) + 1,), math.nan, dtype=dt, device=DEV)
    weight = base[1:].view(V, D + 2)[:, :D]
    weight.copy_(torch.randn(V, D, generator=g))
    tokens = torch.randint(0, V, (M,), generator=g)
    y = myelin.token_embedding(tokens.to(DEV), weight, scale=0.5)
    assert torch.equal(y, _want(tokens.to(DEV), weight, 0.5, None))
    behind = torch.full((M * D + 1,), math.nan, dtype=dt, device=DEV)
    gy = behind[1:].view(M, D)
    gy.copy_(torch.randint(-2, 3, (M, D), generator=g))
    want = torch.zeros(V, D, dtype=torch.float64)
    want.index_add_(0, tokens, gy.cpu().double())
    gw = _grad(tokens.to(DEV), weight, gy, scale=1.0)
    assert torch.equal(gw.cpu(), want.to(dt))
    # the entry points write no more than their rows
    lib_out = torch.full((M * D + 2,), 7.0, dtype=dt, device=DEV)
    grad_out = torch.full((V * D + 2,), 7.0, dtype=dt, device=DEV)
    on = tokens.to(DEV)
    need = _lib.load().myelin_token_embedding_bwd_workspace_bytes(M, V, D)
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device=DEV)
    size, s = lib_out.element_size(), torch.cuda.current_stream().cuda_stream
    _lib.call("myelin_token_embedding", on.data_ptr(), weight.data_ptr(), _lib.DT[dt], D + 2, lib_out.data_ptr() + size,
              M, V, D, 0.5, -(2**63), s)
    _lib.call("myelin_token_embedding_bwd", on.data_ptr(), gy.data_ptr(), _lib.DT[dt], grad_out.data_ptr() + size, M, V,
              D, 1.0, -(2**63), ws.data_ptr(), need, s)
    assert torch.equal(lib_out[1:-1].view(M, D), y) and torch.equal(grad_out[1:-1].view(V, D), gw)
    for t in (lib_out, grad_out):
        assert float(t[0]) == 7.0 and float(t[-1]) == 7.0
