"""Token log probabilities, entropy and alternatives against the f64 oracle."""

import ctypes
import math

import numpy as np
import pytest
import torch

from oracle import logprobs as olp


def test_oracle_rules():
    x = np.array([[1.0, 3.0, 3.0, -np.inf], [-np.inf] * 4, [0.0, np.nan, 9.0, np.nan]])
    lp, ent, top, ids, _ = olp.token_logprobs(x, [0, 2, 2], 4)
    z = 2 + math.exp(-2)
    assert np.isclose(lp[0], -2 - math.log(z)) and lp[1] == -np.inf and np.isnan(lp[2])
    p = np.array([math.exp(-2), 1, 1]) / z
    assert np.isclose(ent[0], -(p * np.log(p)).sum()) and ent[1] == 0 and np.isnan(ent[2])
    assert ids.tolist() == [[1, 2, 0, 3], [0, 1, 2, 3], [1, 3, 2, 0]]
    assert top[0, 3] == -np.inf
    assert olp.token_logprobs(x[:1], [-1], 0)[0][0] == -np.inf


def test_refusals():
    from skinny_mlx_b200 import _lib
    from skinny_mlx_b200.logprobs import token_logprobs

    with pytest.raises(ValueError, match="CUDA"):
        token_logprobs(torch.zeros(2, 8), torch.zeros(2, dtype=torch.int32))
    L, f = _lib.lib(), 0x10000  # (a pointer that is never touched)

    def call(logits=f, ld=64, kind=0, rows=2, v=64, tokens=f, top=4, lp=f, ent=f, tl=f, ti=f, ws=f, n=1 << 30):
        return L.skinny_token_logprobs(logits, ld, kind, rows, v, tokens, top, lp, ent, tl, ti, ws, n, None)

    for kw, status in ((dict(logits=None), -1), (dict(tokens=None), -1), (dict(lp=None), -1), (dict(ent=None), -1),
                       (dict(kind=2), -1), (dict(tl=None), -1), (dict(ti=None), -1), (dict(rows=0), -2), (dict(v=0), -2), (dict(v=2**27 + 1, ld=2**28), -2),
                       (dict(top=33), -2), (dict(top=-1), -2), (dict(v=3, top=4), -2), (dict(ld=63), -2),
                       (dict(logits=f + 1), -4), (dict(logits=f + 2, kind=1), -4), (dict(tokens=f + 2), -4),
                       (dict(ws=None), -5), (dict(n=0), -5), (dict(ws=f + 8), -5)):
        assert call(**kw) == status, kw


@pytest.mark.gpu
def test_python_refusals(cuda_lib, dev):
    from skinny_mlx_b200.logprobs import token_logprobs

    x, t = torch.zeros(2, 8, device=dev), torch.zeros(2, dtype=torch.int32, device=dev)
    for bad in ((x.half(), t, 0), (x[0], t, 0), (x[:, ::2], t, 0), (x, t[:1], 0), (x, t.float(), 0), (x, t.cpu(), 0),
                (x, t, 9), (x, t, -1), (torch.zeros(2, 40, device=dev), t, 33), (x[:, :0], t, 0)):
        with pytest.raises(ValueError):
            token_logprobs(*bad)
    r = token_logprobs(x[:0], t[:0], 3)
    assert r.logprobs.shape == (0,) and r.top_ids.shape == (0, 3)


def _check(x: torch.Tensor, tokens, top_n: int):
    """x on the device; compares with the oracle."""
    from skinny_mlx_b200.logprobs import token_logprobs

    got = token_logprobs(x, tokens, top_n)
    rows, V = x.shape
    lp, ent, top, ids, spread = olp.token_logprobs(x.float().cpu().numpy(), tokens.cpu().numpy(), top_n)
    assert torch.equal(got.top_ids.cpu().long(), torch.from_numpy(ids))
    big = np.nan_to_num(np.abs(np.where(np.isfinite(x.float().cpu().numpy()), x.float().cpu().numpy(), 0)).max(1))
    # Z and sum e (x - m) are sums of terms of one sign, at most V / 256 + 64 of them in a chain, so each is
    # off by (V / 256 + 64) 2^-24 of itself; a term e^d carries 2^-22 from exp2 and 2 |d| 2^-24 from its
    # argument (mean |d| = spread); logprob = (x - m) - ln Z rounds values up to 2 big + ln V four times
    eps = (V / 256 + 64 + 4 + 2 * spread) * 2.0 ** -24
    size = 4 * (2 * big + math.log(V) + 1) * 2.0 ** -24
    for g, want, tol in ((got.logprobs, lp, eps + size), (got.top_logprobs, top, (eps + size)[:, None]),
                         (got.entropy, ent, 2 * eps * (1 + 2 * spread) + size)):
        g = g.cpu().double().numpy()
        fin = np.isfinite(want)
        assert np.array_equal(np.isnan(g), np.isnan(want))
        assert np.array_equal(g[~fin & ~np.isnan(want)], want[~fin & ~np.isnan(want)])
        err = np.abs(np.where(fin, g, 0) - np.where(fin, want, 0))
        assert (err <= tol).all(), (err.max(), np.asarray(tol).min())
    return got


DTYPES = [torch.bfloat16, torch.float32]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,v,top", [(1, 151936, 20), (16, 151936, 5), (3, 151935, 32), (1, 1, 1), (2, 5, 5),
                                        (1, 33, 32), (5, 1000, 0), (300, 777, 7), (40, 4097, 20), (700, 2048, 1),
                                        (9, 50257, 32), (1, 8191, 0), (150, 32000, 32)])
def test_values(cuda_lib, dev, rows, v, top, dtype):
    torch.manual_seed(rows * 31 + v)
    x = (torch.randn(rows, v, device=dev) * 3).to(dtype)
    _check(x, torch.randint(0, v, (rows,), device=dev, dtype=torch.int32), top)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,v", [(450, 98309), (887, 65536)])
def test_many_rows_of_a_large_vocabulary(cuda_lib, dev, rows, v):
    torch.manual_seed(rows)
    x = (torch.randn(rows, v, device=dev) * 3).bfloat16()
    x[3, 40000:] = -math.inf  # (parts with nothing in them)
    x[4, :60000] = -math.inf
    _check(x, torch.randint(0, v, (rows,), device=dev, dtype=torch.int32), 0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("off,ld", [(0, 1003), (1, 1001), (3, 1024), (7, 1000)])
def test_strided_and_unaligned_rows(cuda_lib, dev, off, ld, dtype):
    torch.manual_seed(ld)
    flat = (torch.randn(12 * ld + off, device=dev) * 2).to(dtype)
    x = flat[off:].as_strided((12, 993), (ld, 1), off)
    _check(x, torch.randint(0, 993, (12,), device=dev), 11)  # (int64 ids)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [40, 6000, 151936])
def test_orders_that_defeat_a_threshold(cuda_lib, dev, v, dtype):
    """Constant rows (every value a tie), rows in ascending and descending order, two values only, rows whose
    largest values stand together, at the end, or repeat."""
    x = torch.zeros(9, v, device=dev)
    x[1] = torch.arange(v, device=dev) * (20.0 / v)
    x[2] = -x[1]
    x[3, ::3] = 1.0
    x[4, v - min(v, 35):] = 5.0
    x[5, :30] = torch.arange(30, device=dev) * 0.25
    x[6, v // 2:] = 3.0
    x[7] = torch.arange(v, device=dev) % 17
    x[8, -1] = 1e4
    _check(x.to(dtype), torch.tensor([0, v - 1, 0, 3, v - 1, 29, v // 2, 16, 0], dtype=torch.int32, device=dev), 32)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [70, 20000])
def test_special_values(cuda_lib, dev, v, dtype):
    inf, low = math.inf, torch.finfo(dtype).min
    torch.manual_seed(v)
    x = torch.randn(16, v, device=dev).to(dtype)
    x[0] = -inf                       # nothing left: logprob -inf, entropy 0
    x[1] = -inf
    x[1, 65] = 2.0                    # one token left
    x[2, ::2] = -inf
    x[3] = low                        # the type's lowest value as a mask, of everything
    x[4, 1:] = low
    x[5, 3] = math.nan
    x[6, 66] = inf
    x[7] = math.nan
    x[8, ::2] = -0.0                  # -0 and 0 are one value
    x[8, 1::2] = 0.0
    x[9] = low
    x[9, 60] = low / 2
    x[10] = torch.finfo(dtype).max
    x[11, :] = -inf
    x[11, 5:30] = 1.0                 # fewer tokens left than alternatives asked for
    x[12, 40] = torch.finfo(dtype).max
    x[13, 0] = -inf
    x[14, 0] = inf
    x[14, 1] = -inf
    x[15, 69] = math.nan
    x[15, 68] = inf
    tok = torch.tensor([0, 65, 2, 5, 1, 4, 5, 0, 1, 60, 7, 5, 40, 0, 1, 0], dtype=torch.int32, device=dev)
    _check(x, tok, 32)


@pytest.mark.gpu
@pytest.mark.parametrize("top", [0, 3])
def test_more_rows_than_a_grid_holds(cuda_lib, dev, top):
    torch.manual_seed(1)
    x = torch.randn(70001, 24, device=dev)
    _check(x, torch.randint(0, 24, (70001,), device=dev), top)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [2, 450])
def test_masked_vocabularies(cuda_lib, dev, rows, dtype):
    """Rows of which a mask leaves one, a few, a run, or fewer tokens than alternatives asked for (in one part per
    row and in several)."""
    torch.manual_seed(rows)
    v = 20000
    x = (torch.randn(rows, v, device=dev) * 3).to(dtype)
    keep = torch.zeros(rows, v, dtype=torch.bool, device=dev)
    for r in range(rows):
        n = (1, 7, 19, 20, 21, 300)[r % 6]
        if r % 2:
            keep[r, torch.randperm(v, device=dev)[:n]] = True
        else:
            keep[r, v - 1 - n:v - 1] = True
    x.masked_fill_(~keep, -math.inf if rows == 2 else torch.finfo(dtype).min)
    _check(x, torch.randint(0, v, (rows,), device=dev), 20)


@pytest.mark.gpu
def test_tokens_outside_the_vocabulary(cuda_lib, dev):
    x = torch.randn(6, 100, device=dev)
    tok = torch.tensor([-1, 100, 99, 0, 2**31 - 1, -2**31], device=dev)
    got = _check(x, tok, 0)
    assert got.logprobs.isinf().tolist() == [True, True, False, False, True, True]
    assert token64(x, 2**40) == -math.inf and token64(x, -2**40) == -math.inf


def token64(x, t):
    from skinny_mlx_b200.logprobs import token_logprobs

    return float(token_logprobs(x[:1], torch.tensor([t], device=x.device)).logprobs[0])


@pytest.mark.gpu
def test_streams_graphs_and_repeats(cuda_lib, dev):
    """The same bits from a repeated call, another stream, and two captured graphs replayed together."""
    from skinny_mlx_b200.logprobs import token_logprobs

    torch.manual_seed(3)
    xs = [(torch.randn(4, 151936, device=dev) * 2).to(torch.bfloat16) for _ in range(2)]
    tok = torch.randint(0, 151936, (4,), device=dev, dtype=torch.int32)
    want = [token_logprobs(x, tok, 20) for x in xs]
    again = [token_logprobs(x, tok, 20) for x in xs]
    side = [torch.cuda.Stream(dev) for _ in xs]
    for s in side:
        s.wait_stream(torch.cuda.current_stream(dev))
    other = []
    for s, x in zip(side, xs):
        with torch.cuda.stream(s):
            other.append([token_logprobs(x, tok, 20) for _ in range(20)][-1])
    torch.cuda.synchronize()
    graphs = []
    for s, x in zip(side, xs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side[0]):
            r = token_logprobs(x, tok, 20)
        graphs.append((g, r))
    for _ in range(30):
        for s, (g, _) in zip(side, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for i in range(2):
        for r in (again[i], other[i], graphs[i][1]):
            assert all(torch.equal(a, b) for a, b in zip(want[i], r))
