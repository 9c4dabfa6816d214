"""Paged cache append and attention against the f64 oracle."""

import math

import pytest
import torch

from oracle import paged as opaged

F8 = torch.float8_e4m3fn


def test_oracle_attention_is_a_softmax():
    """One sequence, pages in order: the oracle equals torch's softmax over the causal scores."""
    torch.manual_seed(0)
    q, k, v = torch.randn(1, 3, 4, 64), torch.randn(5, 2, 4, 64), torch.randn(5, 2, 4, 64)
    o, lse, spread, dots, bad = opaged.attention(q, k, v, torch.arange(5)[None].int(), [14], None)
    kk, vv = (x.transpose(1, 2).reshape(20, 2, 64).double().repeat_interleave(2, 1) for x in (k, v))
    for t in range(3):
        s = torch.einsum("hd,jhd->hj", q[0, t].double(), kk[:15 + t]) / 8
        assert torch.allclose(o[0, t], torch.einsum("hj,jhd->hd", s.softmax(-1), vv[:15 + t]))
        assert torch.allclose(lse[0, t], s.logsumexp(-1))
    assert not bad and (spread >= o.abs() - 1e-12).all() and (dots > 0).all()
    # window 1: a token sees itself; idle slots and sequences out of range see nothing
    o, lse, *_ = opaged.attention(q, k, v, torch.arange(5)[None].int(), [14], None, window=1)
    assert torch.allclose(o[0, 1], vv[15])
    assert opaged.attention(q, k, v, torch.arange(5)[None].int(), [14], [0])[1].eq(-math.inf).all()
    assert opaged.attention(q, k, v, torch.arange(5)[None].int(), [18], None)[4]
    assert opaged.attention(q, k, v, torch.tensor([[0, 1, 5, 3, 4]]).int(), [14], None)[4]


# ---------------------------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------------------------
F = 0x10000  # a pointer that is never touched


def _strides(*s):
    import ctypes

    return (ctypes.c_longlong * 3)(*s)


def _append_status(**kw):
    from skinny_mlx_b200 import _lib

    a = dict(q=F, qs=_strides(512, 512, 128), k=F, ks=_strides(256, 256, 128), v=F, vs=_strides(256, 256, 128), qo=F, kp=F,
             vp=F, kps=2 * 16 * 128, vps=2 * 16 * 128, kv=0, ksc=None, vsc=None, table=F, ts=4, width=4, n=9, page=16,
             lengths=F, counts=None, inv=F, rot=32, B=2, T=1, Hq=4, Hkv=2, D=128, stream=None)
    a.update(kw)
    return _lib.lib().skinny_paged_append(*a.values())


def _attn_status(**kw):
    from skinny_mlx_b200 import _lib

    a = dict(q=F, qs=_strides(512, 512, 128), kp=F, vp=F, kps=2 * 16 * 128, vps=2 * 16 * 128, kv=0, ksc=None, vsc=None,
             table=F, ts=4, width=4, n=9, page=16, lengths=F, counts=None, scale=0.1, window=0, out=F, lse=F, B=2, T=1, Hq=4,
             Hkv=2, D=128, ws=F, wsn=1 << 40, stream=None)
    a.update(kw)
    return _lib.lib().skinny_paged_attn(*a.values())


COMMON = [(dict(kp=None), -1), (dict(vp=None), -1), (dict(kv=2), -1), (dict(kv=1), -1), (dict(kv=1, ksc=F), -1),
          (dict(Hkv=0), -2), (dict(D=96), -2), (dict(kps=2 * 16 * 128 - 128), -1), (dict(vps=2 * 16 * 128 + 8), -4),
          (dict(kp=F + 8), -4), (dict(table=None), -1), (dict(lengths=None), -1), (dict(B=0), -2), (dict(B=8193), -2),
          (dict(page=0, kps=1 << 20, vps=1 << 20), -2), (dict(n=0), -2), (dict(width=0), -2), (dict(width=1 << 27, ts=1 << 27), -2),
          (dict(ts=3), -1), (dict(table=F + 2), -4), (dict(counts=F + 1), -4), (dict(q=F + 8), -4),
          (dict(qs=_strides(512, 516, 128)), -4), (dict(qs=None), -1)]


@pytest.mark.parametrize("kw,status", COMMON + [
    (dict(k=None), -1), (dict(v=None), -1), (dict(qo=None), -1), (dict(inv=None), -1), (dict(rot=24), -2),
    (dict(rot=144), -2), (dict(rot=-16), -2), (dict(Hq=0), -2), (dict(T=0), -2), (dict(T=1 << 30), -2), (dict(qo=F + 8), -4),
    (dict(k=F + 2), -4), (dict(vs=_strides(256, 256, 100)), -4)])
def test_append_entry_refuses(kw, status):
    assert _append_status(**kw) == status


@pytest.mark.parametrize("kw,status", COMMON + [
    (dict(q=None), -1), (dict(out=None), -1), (dict(window=-1), -1), (dict(T=0), -3), (dict(T=17), -3), (dict(Hq=3), -2),
    (dict(Hq=0), -2), (dict(Hq=2 * 1025), -2), (dict(n=1 << 30), -2), (dict(vps=1 << 40), -2), (dict(out=F + 8), -4), (dict(lse=F + 2), -4), (dict(ws=None), -5), (dict(wsn=0), -5), (dict(ws=F + 4), -5)])
def test_attention_entry_refuses(kw, status):
    assert _attn_status(**kw) == status


@pytest.mark.parametrize("status", [_append_status, _attn_status])
def test_positions_up_to_the_last_tile_are_32_bit(status):
    """A table whose last tile of keys would end beyond 2^31 is refused."""
    for width, page in (((1 << 27) - 1, 16), ((1 << 31) - 4095, 1), ((1 << 25) - 63, 64)):
        assert status(width=width, ts=width, page=page, kps=1 << 20, vps=1 << 20) == -2


@pytest.mark.parametrize("status", [_append_status, _attn_status])
@pytest.mark.parametrize("kw", [dict(ksc=F), dict(vsc=F), dict(ksc=F, vsc=F)])
def test_scales_of_16_bit_pages_are_refused(status, kw):
    """(The join of split items would apply them, items that one CTA has whole would not.)"""
    assert status(**kw) == -1


def test_workspace_of_unsupported_shapes_is_zero():
    from skinny_mlx_b200 import _lib

    ws = _lib.lib().skinny_paged_attn_workspace_bytes
    for bad in ((0, 1, 4, 2, 128), (8193, 1, 4, 2, 128), (1, 17, 4, 2, 128), (1, 1, 4, 3, 128), (1, 1, 4, 2, 96), (1, 1, 0, 2, 64),
                (1, 1, 2050, 2, 64)):
        assert ws(*bad) == 0


def test_cpu_tensors_are_refused():
    from skinny_mlx_b200 import paged

    x, i = torch.zeros(2, 1, 2, 64, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int32)
    pool = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        paged.attention(x, pool, pool, i[:, None], i)
    with pytest.raises(ValueError, match="CUDA"):
        paged.append(x, x, x, pool, pool, i[:, None], i)


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
class Case:
    """A pool, a table of shuffled pages and a step's inputs on the device."""

    def __init__(self, dev, lengths, counts=None, T=1, Hq=4, Hkv=2, D=128, page=16, kv=torch.bfloat16, seed=0, spare=3,
                 gap=0, gated=False, width=None, std=1.0):
        gen = torch.Generator().manual_seed(seed)
        B = len(lengths)
        self.B, self.T, self.Hq, self.Hkv, self.D, self.page, self.kv, self.dev = B, T, Hq, Hkv, D, page, kv, dev
        self.width = width or max(1, max(-(-(n + T) // page) for n in lengths))
        self.n_pages = B * self.width + spare
        self.table = torch.randperm(self.n_pages, generator=gen)[:B * self.width].view(B, -1).int().to(dev)
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device=dev)
        self.counts = None if counts is None else torch.tensor(counts, dtype=torch.int32, device=dev)
        per = 2 * D if gated else D
        row = (torch.randn(B, T, Hq * per + 2 * Hkv * D, generator=gen) * std).bfloat16().to(dev)
        self.q = row[..., :Hq * per].unflatten(-1, (Hq, per))[..., :D]
        self.k = row[..., Hq * per:Hq * per + Hkv * D].unflatten(-1, (Hkv, D))
        self.v = row[..., Hq * per + Hkv * D:].unflatten(-1, (Hkv, D))
        pages = []
        self.scales = {"k_scale": None, "v_scale": None}
        for name in self.scales:
            x = torch.randn(self.n_pages, Hkv * page * D + gap * D, generator=gen) * std
            if kv == F8:
                self.scales[name] = (0.01 + 0.03 * torch.rand(Hkv, generator=gen)).to(dev)
                x = (x / 0.025).clamp(-448, 448)
            x = x.to(kv).to(dev)
            pages.append(x[:, :Hkv * page * D].unflatten(1, (Hkv, page, D)))
        self.kp, self.vp = pages

    def args(self):
        return self.kp, self.vp, self.table, self.lengths

    def attend(self, **kw):
        from skinny_mlx_b200 import paged

        return paged.attention(self.q, *self.args(), counts=self.counts, return_lse=True, **self.scales, **kw)

    def oracle(self, **kw):
        cpu = lambda x: None if x is None else x.cpu()
        wide = lambda x: x.float().cpu() if x.dtype == F8 else x.cpu()
        return opaged.attention(self.q.cpu(), wide(self.kp), wide(self.vp), self.table.cpu(), self.lengths.cpu(),
                                cpu(self.counts), **{n: cpu(s) for n, s in self.scales.items()}, **kw)


def check_attention(got, want, D):
    """o: the result's rounding to bf16 (2^-8 of it), the probabilities' rounding to 16 bits (2^-8 of
    sum p |v|), and the scores' error: a dot product of D terms in f32, accumulated by the tensor core with
    truncation (2^-22 of sum |q k| per step of 16 terms and 2^-23 per join) is off by e = (D / 8 + 8) 2^-23 dots,
    which changes each p by at most 4 e of itself; f32 sums of p and p v add 2^-16.  lse is off by e, its own
    f32 rounding and the sum of the exponentials (2^-17)."""
    o, lse, spread, dots, _ = want
    go, gl = got[0].double().cpu(), got[1].double().cpu()
    e = (D / 8 + 8) * 2.0 ** -23 * dots
    seen = lse > -math.inf
    assert torch.equal(gl > -math.inf, seen)
    tol = 2.0 ** -8 * o.abs() + (2.0 ** -8 + 2.0 ** -16 + 4 * e[..., None]) * spread * (1 + 2.0 ** -8) + 1e-30
    err = (go - o).abs()
    assert (err <= tol).all(), f"o off by {float((err / tol).max()):.3f} of its tolerance"
    assert (go[~seen] == 0).all()
    err = (gl - lse).abs()[seen]
    tol = (e + 2.0 ** -17 + 2.0 ** -22 * lse.abs())[seen]
    assert (err <= tol).all(), f"lse off by {float((err / tol).max()):.3f} of its tolerance"


# ---------------------------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------------------------
def check_append(c: Case, inv, with_q=True):
    from skinny_mlx_b200 import paged

    before = [c.kp.clone(), c.vp.clone()]
    got = paged.append(c.q if with_q else None, c.k, c.v, *c.args(), inv, counts=c.counts, **c.scales)
    cpu = lambda x: None if x is None else x.cpu()
    q, writes, bad = opaged.append(cpu(c.q), cpu(c.k), cpu(c.v), cpu(c.table), cpu(c.lengths), cpu(c.counts), cpu(inv), c.page,
                                   c.n_pages, **{n: cpu(s) for n, s in c.scales.items()})
    assert bool(paged.device_errors(c.dev, clear=True)) == bad
    # a rotated pair x c - y s in f32: c and s off by at most 2^-22, three roundings: (|x| + |y|) 2^-20
    h = 0 if inv is None else inv.numel()

    def size(x):  # |x| + |its partner|
        a = x.double().abs().cpu()
        if h:
            s = a[..., :h] + a[..., h:2 * h]
            a = torch.cat([s, s, a[..., 2 * h:]], -1)
        return a

    if with_q:
        assert got.shape == c.q.shape and got.is_contiguous()
        err = (got.cpu().double() - q).abs()
        assert (err <= 2.0 ** -8 * q.abs() + 2.0 ** -20 * size(c.q)).all()
    else:
        assert got is None
    # e4m3: half a step is 2^-4 of the value, 2^-10 below the smallest normal number
    half = 2.0 ** -8 if c.kv != F8 else 2.0 ** -4
    least = 0 if c.kv != F8 else 2.0 ** -10
    mask = torch.zeros(c.n_pages, c.page, dtype=torch.bool)
    for pid, slot, kr, vr in writes:
        mask[pid, slot] = True
    pages = [x.float().cpu().double() for x in (c.kp, c.vp)]
    ks = 1.0 if c.scales["k_scale"] is None else c.scales["k_scale"].cpu().double()[:, None]
    big = float(size(c.k).max())
    for pid, slot, kr, vr in writes:
        for x, want, slack in ((pages[0][pid, :, slot], kr, 2.0 ** -20 * big / ks), (pages[1][pid, :, slot], vr, 0)):
            if c.kv == F8:
                want = want.clamp(-448, 448)
            assert ((x - want).abs() <= half * want.abs() + least + slack).all()
    for old, new in zip(before, (c.kp, c.vp)):  # nothing else was touched
        same = (old.view(torch.uint8) == new.view(torch.uint8)) if c.kv == F8 else (old.view(torch.int16) == new.view(torch.int16))
        assert same.cpu().all(-1).transpose(1, 2)[~mask].all()
    return got


def inv_freq(dev, rot, theta=1e6):
    return theta ** (-torch.arange(rot // 2, device=dev, dtype=torch.float32) / (rot // 2))


@pytest.mark.gpu
@pytest.mark.parametrize("kv", [torch.bfloat16, F8])
@pytest.mark.parametrize("D,rot,Hq,Hkv,page,T", [(128, 32, 16, 4, 16, 1), (128, 128, 40, 8, 64, 3), (64, 64, 3, 1, 7, 5),
                                                 (256, 16, 4, 2, 1, 2), (256, 256, 2, 2, 33, 20), (64, 0, 1, 1, 8, 1),
                                                 (128, 96, 5, 5, 24, 130)])
def test_append_values(cuda_lib, dev, kv, D, rot, Hq, Hkv, page, T):
    c = Case(dev, [0, 5, 63, 200], T=T, Hq=Hq, Hkv=Hkv, D=D, page=page, kv=kv, seed=D + T)
    check_append(c, inv_freq(dev, rot) if rot else None)


@pytest.mark.gpu
@pytest.mark.parametrize("kv", [torch.bfloat16, F8])
def test_append_ragged_batch_with_idle_slots(cuda_lib, dev, kv):
    c = Case(dev, [0, 17, 40, 8, 300], counts=[4, 0, 1, 3, 4], T=4, kv=kv, page=16, gated=True, gap=5)
    check_append(c, inv_freq(dev, 32))
    c = Case(dev, [3], counts=[0], T=2, kv=kv)
    assert (check_append(c, inv_freq(dev, 32)) == 0).all()
    check_append(Case(dev, [3, 9], T=2, kv=kv), inv_freq(dev, 64), with_q=False)


@pytest.mark.gpu
def test_append_far_positions(cuda_lib, dev):
    """Positions whose angle an f32 product would not hold."""
    c = Case(dev, [1_048_570, 131_071, 16_777_217], T=4, page=64, width=4)
    c.table = torch.zeros(3, (16_777_300 // 64), dtype=torch.int32, device=dev)
    for b, n in enumerate((1_048_570, 131_071, 16_777_217)):
        c.table[b, n // 64:(n + 3) // 64 + 1] = torch.arange(3 * b, 3 * b + (n + 3) // 64 + 1 - n // 64, device=dev).int()
    check_append(c, inv_freq(dev, 128, 1e4))


@pytest.mark.gpu
def test_append_e4m3_special_values(cuda_lib, dev):
    from skinny_mlx_b200 import paged

    c = Case(dev, [0], kv=F8, D=64, Hkv=1, Hq=1)
    x = torch.zeros(64)
    x[:12] = torch.tensor([448.0, 464.0, 465.0, 1e30, -1e30, math.inf, -math.inf, math.nan, 2.0 ** -9, 2.0 ** -10, 2.0 ** -11, -0.0])
    c.k[0, 0, 0] = x.to(dev)
    c.v[0, 0, 0] = x.to(dev)
    one = torch.ones(1, device=dev)
    paged.append(None, c.k, c.v, *c.args(), k_scale=one, v_scale=one)
    want = x.bfloat16().float().clamp(-448, 448).to(F8)
    pid = int(c.table[0, 0])
    for pool in (c.kp, c.vp):
        got = pool[pid, 0, 0].cpu()
        assert torch.equal(got.view(torch.uint8) & 0x7F, want.view(torch.uint8) & 0x7F)
        assert torch.equal(got.float()[:7], want.float()[:7])


@pytest.mark.gpu
@pytest.mark.parametrize("kv", [torch.bfloat16, F8])
def test_what_is_out_of_range_touches_nothing(cuda_lib, dev, kv):
    """Sequences that do not fit their table, bad counts, page ids outside the pool: reported, the rest of the
    batch unharmed.  (Every index is checked in the kernels before it forms an address.)"""
    from skinny_mlx_b200 import paged

    paged.device_errors(dev, clear=True)
    c = Case(dev, [30, 40, 2, 5, 20, 31], T=2, page=16, kv=kv, seed=5, width=3)
    c.lengths = torch.tensor([30, -1, 2, 2**31 - 1, 20, 47], dtype=torch.int32, device=dev)
    c.table[2, 0], c.table[4, 1] = -1, c.n_pages
    check_append(c, inv_freq(dev, 32))
    got = c.attend()
    assert paged.device_errors(dev, clear=True) == 1 << 9
    check_attention(got, c.oracle(), c.D)
    c = Case(dev, [30, 40, 2], counts=[3, -1, 2], T=2, page=16, kv=kv, seed=6)
    check_append(c, inv_freq(dev, 32))
    got = c.attend()
    assert paged.device_errors(dev, clear=True) == 1 << 9
    check_attention(got, c.oracle(), c.D)
    assert paged.device_errors(dev) == 0


# ---------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("kv", [torch.bfloat16, F8])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("Hq,Hkv,T,page", [(4, 4, 1, 16), (8, 2, 1, 64), (10, 2, 1, 24), (8, 1, 1, 1), (6, 2, 3, 7), (16, 1, 2, 48),
                                           (4, 1, 8, 16), (8, 2, 16, 32), (5, 1, 13, 100), (17, 1, 1, 16), (40, 1, 4, 8)])
def test_attention_values(cuda_lib, dev, Hq, Hkv, T, page, D, kv):
    c = Case(dev, [0, 1, 15, 64, 131, 257], T=T, Hq=Hq, Hkv=Hkv, D=D, page=page, kv=kv, seed=Hq + T)
    check_attention(c.attend(), c.oracle(), D)


@pytest.mark.gpu
@pytest.mark.parametrize("kv", [torch.bfloat16, F8])
@pytest.mark.parametrize("window", [1, 2, 16, 17, 100])
@pytest.mark.parametrize("T", [1, 5, 16])
def test_attention_window(cuda_lib, dev, window, T, kv):
    c = Case(dev, [0, 3, 95, 300], T=T, Hq=6, Hkv=2, page=16, kv=kv, seed=window)
    check_attention(c.attend(window=window), c.oracle(window=window), c.D)


@pytest.mark.gpu
@pytest.mark.parametrize("kv", [torch.bfloat16, F8])
def test_attention_ragged_counts_scale_and_strides(cuda_lib, dev, kv):
    c = Case(dev, [0, 17, 400, 8, 90, 0], counts=[4, 0, 1, 3, 4, 0], T=4, Hq=8, Hkv=4, kv=kv, gated=True, gap=7)
    check_attention(c.attend(scale=0.3), c.oracle(scale=0.3), c.D)
    check_attention(c.attend(scale=-0.05), c.oracle(scale=-0.05), c.D)
    # queries whose rows are not aligned, or whose dims are not dense, are copied
    want = c.attend()
    raw = torch.empty(c.q.numel() + 4, dtype=torch.bfloat16, device=dev)
    odd = raw[4:].view(c.q.shape)
    for q in (odd.copy_(c.q), c.q.transpose(2, 3).contiguous().transpose(2, 3), c.q.transpose(0, 1).contiguous().transpose(0, 1)):
        c.q = q
        assert all(torch.equal(a, b) for a, b in zip(c.attend(), want))


@pytest.mark.gpu
@pytest.mark.parametrize("kv", [torch.bfloat16, F8])
@pytest.mark.parametrize("lengths,page,T,Hq,Hkv", [([4096], 64, 1, 16, 4), ([2047], 16, 8, 16, 4), ([9001, 1], 32, 1, 8, 2),
                                                   ([700 + 37 * i for i in range(40)], 16, 1, 8, 2), ([20011], 128, 1, 4, 1),
                                                   ([63 * i for i in range(70)], 16, 2, 2, 2)])
def test_attention_long_and_many(cuda_lib, dev, lengths, page, T, Hq, Hkv, kv):
    c = Case(dev, lengths, T=T, Hq=Hq, Hkv=Hkv, page=page, kv=kv, seed=len(lengths))
    check_attention(c.attend(), c.oracle(), c.D)


@pytest.mark.gpu
@pytest.mark.parametrize("kv", [torch.bfloat16, F8])
@pytest.mark.parametrize("B", [33, 129, 700])
def test_attention_batches_wider_than_a_warp_and_a_block(cuda_lib, dev, B, kv):
    """More sequences than a warp, a CTA's threads, and several per thread; idle ones and empty ones among them."""
    lengths = [(37 * i) % 150 if i % 7 else 0 for i in range(B)]
    counts = [0 if i % 5 == 3 or i < 3 else 1 for i in range(B)]
    c = Case(dev, lengths, counts, T=1, Hq=2, Hkv=1, D=64, page=8, kv=kv, seed=B)
    check_attention(c.attend(), c.oracle(), c.D)
    c.counts = torch.zeros_like(c.counts)
    o, lse = c.attend()
    assert (o == 0).all() and (lse == -math.inf).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kv", [torch.bfloat16, F8])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("page", [2, 3, 4, 8, 12, 16, 31, 32, 96, 1024])
def test_attention_page_sizes(cuda_lib, dev, page, D, kv):
    """Every size of copy a page allows, with windows that begin and lengths that end inside one."""
    c = Case(dev, [0, 45, 262], T=3, Hq=6, Hkv=2, D=D, page=page, kv=kv, seed=page)
    check_attention(c.attend(), c.oracle(), D)
    check_attention(c.attend(window=37), c.oracle(window=37), D)


@pytest.mark.gpu
def test_pages_before_the_window_may_be_gone(cuda_lib, dev):
    """Table entries of pages that no row sees are not looked at."""
    from skinny_mlx_b200 import paged

    c = Case(dev, [300, 97], T=2, Hq=4, Hkv=2, page=16, seed=1)
    want = c.oracle(window=40)
    c.table[0, :(300 + 1 - 40) // 16] = -1
    c.table[1, :(97 + 1 - 40) // 16] = 10 ** 6
    c.table[1, (97 + 2 + 15) // 16:] = -7
    check_attention(c.attend(window=40), want, c.D)
    assert paged.device_errors(dev, clear=True) == 0


@pytest.mark.gpu
def test_calls_from_two_threads(cuda_lib, dev):
    """Two threads with streams of their own: every result is the one of a call alone."""
    import threading

    cases = [Case(dev, [500 + 300 * i, 40, 1200], T=1 + 3 * i, Hq=8, Hkv=2, page=16, seed=i) for i in range(2)]
    want = [c.attend() for c in cases]
    torch.cuda.synchronize()
    bad = []

    def work(c, w):
        with torch.cuda.stream(torch.cuda.Stream(dev)):
            for _ in range(200):
                got = c.attend()
                if not all(torch.equal(a, b) for a, b in zip(got, w)):
                    bad.append(1)

    ts = [threading.Thread(target=work, args=a) for a in zip(cases, want)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert not bad


@pytest.mark.gpu
@pytest.mark.parametrize("B", [3, 40, 300])
def test_a_batch_of_idle_slots(cuda_lib, dev, B):
    c = Case(dev, [17] * B, counts=[0] * B, T=2)
    o, lse = c.attend()
    assert (o == 0).all() and (lse == -math.inf).all()
    check_append(c, inv_freq(dev, 32))


@pytest.mark.gpu
@pytest.mark.parametrize("T,kv", [(1, torch.bfloat16), (16, F8)])
def test_attention_of_a_thousand_heads_per_kv_head(cuda_lib, dev, T, kv):
    c = Case(dev, [100, 3], T=T, Hq=1024, Hkv=1, D=64, kv=kv)
    check_attention(c.attend(), c.oracle(), c.D)


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(window=2**31 - 1), dict(window=300), dict(scale=-0.3), dict(scale=0.0)])
@pytest.mark.parametrize("kv", [torch.bfloat16, F8])
def test_attention_extreme_arguments(cuda_lib, dev, kv, kw):
    c = Case(dev, [250, 0, 77], T=3, kv=kv)
    check_attention(c.attend(**kw), c.oracle(**kw), c.D)


@pytest.mark.gpu
def test_inputs_of_other_orders(cuda_lib, dev):
    """Queries, keys and values laid out head by head, a table that is a slice of a wider one, one sequence
    whose table is an expanded row."""
    c = Case(dev, [60, 9, 33], T=4, Hq=6, Hkv=2, D=128)
    swap = lambda x: x.transpose(1, 2).contiguous().transpose(1, 2)
    c.q, c.k, c.v = swap(c.q), swap(c.k), swap(c.v)
    wide = torch.full((3, c.width + 5), -7, dtype=torch.int32, device=dev)
    wide[:, 2:2 + c.width] = c.table
    c.table = wide[:, 2:2 + c.width]
    check_append(c, inv_freq(dev, 64))
    check_attention(c.attend(), c.oracle(), c.D)
    c = Case(dev, [60], T=4)
    c.table = c.table[0].expand(1, -1)
    check_append(c, None, with_q=False)
    check_attention(c.attend(), c.oracle(), c.D)


@pytest.mark.gpu
def test_attention_sharp_and_large_scores(cuda_lib, dev):
    """Scores far apart (one key takes everything, late or early) and large ones of both signs."""
    c = Case(dev, [200, 333], T=2, Hq=8, Hkv=2, std=6.0, seed=2)
    check_attention(c.attend(), c.oracle(), c.D)
    for at in (0, 100, 198):
        c = Case(dev, [199], T=1, Hq=4, Hkv=1, seed=at)
        c.kp[int(c.table[0, at // 16]), 0, at % 16] = (c.q[0, 0, 1] * 9)
        check_attention(c.attend(), c.oracle(), c.D)


@pytest.mark.gpu
@pytest.mark.parametrize("kv", [torch.bfloat16, F8])
@pytest.mark.parametrize("T,window", [(1, None), (5, None), (5, 20), (16, None)])
def test_what_is_not_seen_has_no_influence(cuda_lib, dev, T, window, kv):
    """NaN and infinities behind the last position, before the window, in pages of nobody, and in later tokens of
    the same draft leave the rows that do not see them as they were."""
    c = Case(dev, [45, 130, 7], T=T, Hq=6, Hkv=2, page=16, kv=kv, seed=T)
    want = c.attend(window=window)
    bad = [math.nan] if kv == F8 else [math.nan, math.inf, -math.inf]
    seen = torch.zeros(c.n_pages, 16, dtype=torch.bool)
    for b, n in enumerate((45, 130, 7)):
        for j in range(max(0, n + 1 - window) if window else 0, n + T):
            seen[int(c.table[b, j // 16]), j % 16] = True
    for x in bad:
        for pool in (c.kp, c.vp):
            pool.transpose(1, 2)[(~seen).to(dev)] = torch.tensor(x, device=dev).to(kv)
        got = c.attend(window=window)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    for t in range(1, T):  # token t's own key and value: rows before it do not change
        for pool, x in ((c.kp, bad[0]), (c.vp, bad[-1])):
            for b, n in enumerate((45, 130, 7)):
                pool[int(c.table[b, (n + t) // 16]), :, (n + t) % 16] = torch.tensor(x, device=dev).to(kv)
        got = c.attend(window=window)
        # (two roundings of the result, 2^-7 of it, and of the probabilities, 2^-7 sum p |v|)
        assert all(torch.allclose(a[:, :t].float(), b[:, :t].float(), rtol=2.0 ** -7, atol=2.0 ** -7) for a, b in zip(got, want))
        assert got[0][:, t].isnan().all()
        c = Case(dev, [45, 130, 7], T=T, Hq=6, Hkv=2, page=16, kv=kv, seed=T)


@pytest.mark.gpu
def test_infinite_values_that_are_seen(cuda_lib, dev):
    """An infinite value reaches exactly the dims and the rows that see it."""
    c = Case(dev, [30], T=6, Hq=4, Hkv=2, seed=4)
    pid, slot = int(c.table[0, 33 // 16]), 33 % 16
    c.vp[pid, 1, slot, 5] = math.inf
    o = c.attend()[0].float()
    hit = torch.zeros_like(o, dtype=torch.bool)
    hit[0, 3:, 2:, 5] = True
    assert torch.equal(o.isinf(), hit) and not o.isnan().any()


MANY = [(12, 4, 11, 16), (40, 8, 16, 8), (8, 1, 13, 40), (16, 1, 8, 128), (20, 1, 16, 64)]  # 33, 80, 104, 128, 320 rows


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,Hkv,T,page", MANY)
def test_attention_of_many_rows(cuda_lib, dev, Hq, Hkv, T, page, D):
    """More than 32 rows per kv head: lengths around a tile's end, idle slots, windows, pools with gaps between
    pages of which the odd one allows no copies of whole eights, sharp scores."""
    lengths = [0, 5, 127, 128, 500, 1029, 3, 0]
    counts = [T, 1, T, 2, 0, T, T - 1, 0]
    for kw in (dict(), dict(gap=8), dict(gap=3)):
        c = Case(dev, lengths, counts, T=T, Hq=Hq, Hkv=Hkv, page=page, D=D, seed=Hq + T, **kw)
        check_attention(c.attend(), c.oracle(), D)
    c.q = c.q * 6
    check_attention(c.attend(window=100, scale=-0.2), c.oracle(window=100, scale=-0.2), D)
    check_attention(c.attend(scale=0.0), c.oracle(scale=0.0), D)


@pytest.mark.gpu
@pytest.mark.parametrize("Hq,Hkv,T,page,n", [(12, 4, 11, 16, 9001), (8, 1, 13, 40, 4000), (20, 1, 16, 64, 1500)])
def test_many_rows_of_long_and_many_sequences(cuda_lib, dev, Hq, Hkv, T, page, n):
    c = Case(dev, [n, 2], T=T, Hq=Hq, Hkv=Hkv, page=page, seed=3)
    check_attention(c.attend(), c.oracle(), c.D)
    lengths = [(53 * i) % 300 for i in range(250)]
    c = Case(dev, lengths, [T if i % 8 == 5 else i % 3 == 1 for i in range(250)], T=T, Hq=Hq, Hkv=Hkv, page=page, D=64, seed=4)
    check_attention(c.attend(), c.oracle(), c.D)


@pytest.mark.gpu
@pytest.mark.parametrize("window", [None, 40])
@pytest.mark.parametrize("Hq,Hkv,T,page", MANY)
def test_many_rows_and_what_they_do_not_see(cuda_lib, dev, Hq, Hkv, T, page, window):
    from skinny_mlx_b200 import paged

    lengths = [45, 300, 7]
    c = Case(dev, lengths, T=T, Hq=Hq, Hkv=Hkv, page=page, seed=T)
    want = c.attend(window=window)
    seen = torch.zeros(c.n_pages, page, dtype=torch.bool)
    for b, n in enumerate(lengths):
        for j in range(max(0, n + 1 - window) if window else 0, n + T):
            seen[int(c.table[b, j // page]), j % page] = True
    for x in (math.nan, math.inf, -math.inf):
        for pool in (c.kp, c.vp):
            pool.transpose(1, 2)[(~seen).to(dev)] = x
        assert all(torch.equal(a, b) for a, b in zip(c.attend(window=window), want))
    t = T // 2  # a token's own value: the tokens before it do not change
    for b, n in enumerate(lengths):
        c.vp[int(c.table[b, (n + t) // page]), :, (n + t) % page] = -math.inf
    got = c.attend(window=window)
    # (two roundings of the result, 2^-7 of it, and of the probabilities, 2^-7 sum p |v|)
    assert all(torch.allclose(a[:, :t].float(), b[:, :t].float(), rtol=2.0 ** -7, atol=2.0 ** -7) for a, b in zip(got, want))
    assert (got[0][:, t:] == -math.inf).all()
    # pages of nobody are skipped and reported
    c.table[1, 1] = c.n_pages
    c.table[2, :] = -1
    want = c.oracle(window=window)
    got = c.attend(window=window)
    lse = want[1]
    assert torch.equal(got[1].cpu() > -math.inf, lse > -math.inf) and (got[0][2] == 0).all()
    assert paged.device_errors(dev, clear=True) == 1 << 9


@pytest.mark.gpu
@pytest.mark.parametrize("Hq,Hkv,T,page", MANY)
def test_infinite_values_that_many_rows_see(cuda_lib, dev, Hq, Hkv, T, page):
    """In a tile that every row sees whole, in either half of it."""
    c = Case(dev, [1000], T=T, Hq=Hq, Hkv=Hkv, page=page, seed=4)
    for j, d, x in ((3, 5, math.inf), (100, 77, -math.inf), (200, 0, math.inf), (700, 127, math.nan)):
        c.vp[int(c.table[0, j // page]), Hkv - 1, j % page, d] = x
    o = c.attend()[0].float()
    mine = o[:, :, Hq - Hq // Hkv:]
    assert (mine[..., 5] == math.inf).all() and (mine[..., 77] == -math.inf).all() and (mine[..., 0] == math.inf).all()
    assert mine[..., 127].isnan().all()
    o = o.clone()
    o[:, :, Hq - Hq // Hkv:, [5, 77, 0, 127]] = 0
    assert o.isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("Hkv,D", [(4, 128), (2, 128), (2, 256)])
def test_many_rows_on_two_streams_and_replayed(cuda_lib, dev, Hkv, D):
    """Two batches at a time, eagerly and from graphs whose lengths change between replays: the bits of calls one
    after the other."""
    cases = [Case(dev, [700 + 91 * i, 5, 2000], T=16, Hq=16, Hkv=Hkv, D=D, page=32, seed=i, width=70) for i in range(2)]
    lengths = [[(c.lengths - 3 * n * (c.lengths > 100)).int() for n in range(4)] for c in cases]
    want = []
    for c, ls in zip(cases, lengths):
        want.append([])
        for n in ls:
            c.lengths = n
            want[-1].append(c.attend())
    check_attention(want[1][3], cases[1].oracle(), D)
    streams = [torch.cuda.Stream(dev) for _ in cases]
    for c, ls in zip(cases, lengths):
        c.lengths = ls[0].clone()
    torch.cuda.synchronize()
    graphs = []
    for c, s in zip(cases, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            out = [c.attend() for _ in range(3)]
        graphs.append((g, out))
    for n in range(4):
        eager = []
        for c, ls, s in zip(cases, lengths, streams):
            with torch.cuda.stream(s):
                c.lengths.copy_(ls[n])
                eager.append([c.attend() for _ in range(3)])
        for (g, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for i in range(2):
            for got in eager[i] + graphs[i][1]:
                assert all(torch.equal(x, y) for x, y in zip(got, want[i][n]))


@pytest.mark.gpu
@pytest.mark.parametrize("Hq,Hkv,T,page", MANY)
def test_many_rows_of_wide_heads(cuda_lib, dev, Hq, Hkv, T, page):
    """Heads of 256: values, windows and scales, a longer sequence, and infinities that are seen or not."""
    c = Case(dev, [0, 63, 64, 500, 1029, 3], [T, T, 1, 0, T - 1, 2], T=T, Hq=Hq, Hkv=Hkv, page=page, D=256, seed=Hq, gap=8)
    check_attention(c.attend(), c.oracle(), 256)
    c.q = c.q * 6
    check_attention(c.attend(window=100, scale=-0.2), c.oracle(window=100, scale=-0.2), 256)
    c = Case(dev, [3000], T=T, Hq=Hq, Hkv=Hkv, page=page, D=256, seed=5)
    want = c.attend()
    check_attention(want, c.oracle(), 256)
    c.vp[int(c.table[0, 70 // page]), Hkv - 1, 70 % page, 200] = math.inf  # every row sees it
    j = 3000 + T // 2                                                      # rows from T / 2 on see it
    c.vp[int(c.table[0, j // page]), 0, j % page, 31] = -math.inf
    o = c.attend()[0].float()
    hit = torch.zeros_like(o, dtype=torch.bool)
    hit[:, :, Hq - Hq // Hkv:, 200] = True
    hit[:, T // 2:, :Hq // Hkv, 31] = True
    assert torch.equal(o.isinf(), hit) and not o.isnan().any()
    assert torch.allclose(o[~hit], want[0].float()[~hit], rtol=2.0 ** -7, atol=2.0 ** -7)  # (two roundings, as above)


@pytest.mark.gpu
def test_shared_pages_and_one_page_twice(cuda_lib, dev):
    """Sequences that share a prefix's pages, and a table that names a page twice."""
    c = Case(dev, [70, 90, 64], T=1, Hq=4, Hkv=2, page=16, seed=8)
    c.table[1, :4] = c.table[0, :4]
    c.table[2, 1] = c.table[2, 0]
    check_attention(c.attend(), c.oracle(), c.D)


@pytest.mark.gpu
def test_offsets_beyond_32_bits(cuda_lib, dev):
    """Pages further than 2^32 bytes into a pool, and page strides that pass 2^31 elements in all."""
    torch.manual_seed(0)
    big = torch.empty(5, 1 << 30, dtype=torch.bfloat16, device=dev)  # 10 GB: page 4 starts 2^33 bytes in
    c = Case(dev, [40], T=2, Hq=4, Hkv=2, page=16)
    n = 2 * 16 * 128
    for i, pool in enumerate(("kp", "vp")):
        x = big[:, i * n:(i + 1) * n].unflatten(1, (2, 16, 128))
        x.copy_(torch.randn(5, 2, 16, 128, device=dev))
        setattr(c, pool, x)
    c.n_pages = 5
    c.table = torch.tensor([[4, 0, 3]], dtype=torch.int32, device=dev)
    check_append(c, inv_freq(dev, 32))
    check_attention(c.attend(), c.oracle(), c.D)


@pytest.mark.gpu
def test_step_of_a_batch_streams_and_graphs(cuda_lib, dev):
    """append then attention for several steps, eagerly, on another stream, and replayed from two graphs that
    run side by side: the same bits, and the oracle's values."""
    from skinny_mlx_b200 import paged

    inv = inv_freq(dev, 32)

    def steps(c, n=3):
        outs = []
        for _ in range(n):
            q = paged.append(c.q, c.k, c.v, *c.args(), inv, counts=c.counts, **c.scales)
            outs.append(paged.attention(q, *c.args(), counts=c.counts, return_lse=True, **c.scales))
            c.lengths += c.counts
        return outs

    def case(i):
        return Case(dev, [100 + i, 900, 0, 37], counts=[2, 1, 2, 0], T=2, Hq=8, Hkv=2, page=16, seed=i, width=64)

    want, finals = [], []
    for i in range(2):
        c = case(i)
        want.append(steps(c))
        finals.append(c)
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    torch.cuda.synchronize()
    other = []
    for i, s in enumerate(streams):
        c = case(i)
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            other.append(steps(c))
    torch.cuda.synchronize()
    graphs = []
    for i in range(2):
        c = case(i)
        torch.cuda.synchronize()
        start = (c.lengths.clone(), c.kp.clone(), c.vp.clone())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=streams[0]):
            outs = steps(c)
        graphs.append((g, c, start, outs))
    for _ in range(5):
        for g, c, start, outs in graphs:
            for x, y in zip((c.lengths, c.kp, c.vp), start):
                x.copy_(y)
        torch.cuda.synchronize()
        for s, (g, c, start, outs) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for i in range(2):
            for a, b, d in zip(want[i], other[i], graphs[i][3]):
                assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
                assert torch.equal(a[0], d[0]) and torch.equal(a[1], d[1])
    c = finals[0]
    assert c.lengths.tolist() == [106, 903, 6, 37]
    check_append(c, inv)
    c.q = paged.append(c.q, c.k, c.v, *c.args(), inv, counts=c.counts)
    check_attention(c.attend(), c.oracle(), c.D)


@pytest.mark.gpu
def test_python_refusals(cuda_lib, dev):
    from skinny_mlx_b200 import paged

    c = Case(dev, [5, 9], T=2, Hq=4, Hkv=2)
    ok = dict(q=c.q, k_pages=c.kp, v_pages=c.vp, block_table=c.table, lengths=c.lengths)
    paged.attention(**ok)
    i64 = c.lengths.long()
    for bad in (dict(q=c.q.float()), dict(q=c.q[0]), dict(q=c.q[:1]), dict(q=c.q[..., :64]), dict(q=c.q[:, :, :3]), dict(q=c.q.cpu()),
                dict(k_pages=c.kp.half()), dict(k_pages=c.kp[:, :1]), dict(k_pages=c.kp.transpose(1, 2)), dict(v_pages=c.vp.to(F8)),
                dict(k_pages=c.kp.cpu(), v_pages=c.vp.cpu()), dict(block_table=c.table.long()), dict(block_table=c.table[:1]),
                dict(block_table=c.table[:, :0]), dict(lengths=i64), dict(lengths=c.lengths[:1]), dict(counts=i64),
                dict(counts=c.lengths.cpu()), dict(window=0), dict(k_scale=torch.ones(2, device=dev)),
                dict(k_pages=c.kp.to(F8), v_pages=c.vp.to(F8)), dict(q=c.q.repeat(1, 9, 1, 1))):
        with pytest.raises(ValueError):
            paged.attention(**{**ok, **bad})
    ok = dict(q=c.q, k=c.k, v=c.v, k_pages=c.kp, v_pages=c.vp, block_table=c.table, lengths=c.lengths, inv_freq=inv_freq(dev, 32))
    paged.append(**ok)
    for bad in (dict(k=c.k[:, :, :1]), dict(v=c.v[:, :1]), dict(k=c.k.float()), dict(inv_freq=inv_freq(dev, 20)),
                dict(inv_freq=inv_freq(dev, 256)), dict(inv_freq=inv_freq(dev, 32).double()), dict(inv_freq=inv_freq("cpu", 32))):
        with pytest.raises(ValueError):
            paged.append(**{**ok, **bad})
    # an empty batch and a step of no tokens are calls that do nothing
    assert paged.attention(**{**dict(q=c.q[:, :0], k_pages=c.kp, v_pages=c.vp, block_table=c.table, lengths=c.lengths)}).shape == (2, 0, 4, 128)
    z = dict(block_table=c.table[:0], lengths=c.lengths[:0], k_pages=c.kp, v_pages=c.vp)
    assert paged.attention(q=c.q[:0], **z).shape == (0, 2, 4, 128)
    assert paged.append(c.q[:0], c.k[:0], c.v[:0], **z).shape == (0, 2, 4, 128)
    assert paged.device_errors(dev) == 0


# ---------------------------------------------------------------------------------------------
# keys that take nearly all of a row
# ---------------------------------------------------------------------------------------------
def _sink(dev, kv, T, lengths, at, nats, **kw):
    """Sequences in which the key at position at(length), of value 0, lies `nats` above all others for every row
    (scale 1): dim 0 of the queries is 8 and of the other keys 0, the other dims give scores of some +-0.5."""
    c = Case(dev, lengths, T=T, kv=kv, std=0.2, **kw)
    ks = torch.ones(c.Hkv) if c.scales["k_scale"] is None else c.scales["k_scale"].cpu()
    c.q = c.q.clone()
    c.q[..., 0] = 8
    c.kp[..., 0] = 0
    for b, n in enumerate(lengths):
        j = at(n)
        pid = int(c.table[b, j // c.page])
        for h in range(c.Hkv):
            c.kp[pid, h, j % c.page] = 0
            c.kp[pid, h, j % c.page, 0] = (nats / 8 / ks[h]).to(kv).to(dev)
        c.vp[pid, :, j % c.page] = 0
    return c


@pytest.mark.gpu
@pytest.mark.parametrize("kv", [torch.bfloat16, F8])
@pytest.mark.parametrize("T", [1, 8, 16])
@pytest.mark.parametrize("nats", [10, 14, 16, 17, 18, 20, 22, 25, 40])
def test_one_key_takes_nearly_all(cuda_lib, dev, T, nats, kv):
    """First, in the middle, last: what the other keys add keeps its relative precision however little it is.  (The
    bounds are check_attention's: each p is off by half a bf16 step, 2^-8 of itself, whatever its size.)"""
    for at in (lambda n: 0, lambda n: n // 2, lambda n: n - 1):
        c = _sink(dev, kv, T, [1500, 300, 40], at, nats, Hq=8, Hkv=2, page=16, seed=nats)
        check_attention(c.attend(scale=1.0), c.oracle(scale=1.0), c.D)


@pytest.mark.gpu
@pytest.mark.parametrize("D,Hq,Hkv", [(64, 2, 2), (64, 16, 1), (256, 2, 1), (256, 16, 1)])
def test_one_key_takes_nearly_all_of_other_heads(cuda_lib, dev, D, Hq, Hkv):
    for T in (1, 4):
        c = _sink(dev, F8, T, [1500, 300, 40], lambda n: 0, 20, Hq=Hq, Hkv=Hkv, D=D, page=32, seed=D)
        check_attention(c.attend(scale=1.0), c.oracle(scale=1.0), D)


@pytest.mark.gpu
@pytest.mark.parametrize("kv", [torch.bfloat16, F8])
@pytest.mark.parametrize("power", [10, 16, 26, 60, 120])
def test_query_elements_far_apart(cuda_lib, dev, power, kv):
    """One element of a query row is 2^power and meets keys that are 0 there: the others keep their precision.
    The same with an infinity, which gives NaN in its own row alone."""
    c = Case(dev, [300, 40], T=3, Hq=4, Hkv=2, kv=kv, seed=power)
    c.q = c.q.clone()
    c.q[:, :, 1::2, 5] = 2.0 ** power
    c.kp[..., 5] = 0
    check_attention(c.attend(), c.oracle(), c.D)
    want = c.attend()[0]
    c.q[:, 1, 1, 5] = math.inf
    got = c.attend()[0]
    assert got[:, 1, 1].isnan().all()
    got[:, 1, 1] = want[:, 1, 1]
    assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("Hq,Hkv,T,page,D", [(8, 1, 13, 40, 128), (20, 1, 16, 16, 128), (16, 1, 8, 8, 64), (8, 1, 16, 16, 256),
                                             (12, 4, 11, 16, 128), (8, 2, 3, 16, 128), (4, 2, 1, 16, 64)])
def test_infinite_values_beside_a_page_that_is_skipped(cuda_lib, dev, Hq, Hkv, T, page, D):
    """A page id outside the pool in the middle of a context, infinities and NaN in the tile around it: only the
    page is skipped, every row gets what it sees of the others."""
    from skinny_mlx_b200 import paged

    paged.device_errors(dev, clear=True)
    c = Case(dev, [1000, 400], T=T, Hq=Hq, Hkv=Hkv, page=page, D=D, seed=9)
    c.table[0, 160 // page] = c.n_pages  # keys 160 to 160 + page
    want = c.oracle()
    for j, d, x in ((150, 5, math.inf), (155, 33, -math.inf), (210, 9, math.nan), (1000, 40, math.inf)):
        c.vp[int(c.table[0, j // page]), Hkv - 1, j % page, d] = x
    got = c.attend()
    assert paged.device_errors(dev, clear=True) == 1 << 9
    o = got[0].float()
    mine = o[0, :, Hq - Hq // Hkv:]
    assert (mine[..., 5] == math.inf).all() and (mine[..., 33] == -math.inf).all() and mine[..., 9].isnan().all()
    assert (mine[..., 40] == math.inf).all()
    got[0][0, :, Hq - Hq // Hkv:, [5, 9, 33, 40]] = 0
    for x in (want[0], want[2]):
        x[0, :, Hq - Hq // Hkv:, [5, 9, 33, 40]] = 0
    check_attention(got, want, D)


@pytest.mark.gpu
def test_pools_of_nothing_are_refused(cuda_lib, dev):
    from skinny_mlx_b200 import paged

    c = Case(dev, [5, 9], T=2, Hq=4, Hkv=2)
    for cut in (lambda x: x[:0], lambda x: x[:, :, :0], lambda x: x[:1, :, :0]):
        with pytest.raises(ValueError):
            paged.attention(c.q, cut(c.kp), cut(c.vp), c.table, c.lengths)
        with pytest.raises(ValueError):
            paged.append(c.q, c.k, c.v, cut(c.kp), cut(c.vp), c.table, c.lengths)
    none = [x[:, :0] for x in (c.kp, c.vp)]
    with pytest.raises(ValueError):
        paged.attention(c.q, *none, c.table, c.lengths)
    with pytest.raises(ValueError):
        paged.append(None, c.k[:, :, :0], c.v[:, :, :0], *none, c.table, c.lengths)


@pytest.mark.gpu
@pytest.mark.parametrize("D,Hq,T", [(64, 1, 1), (128, 4, 1), (256, 2, 4), (128, 4, 5)])
def test_every_e4m3_number_as_key_and_value(cuda_lib, dev, D, Hq, T):
    """Each of the 256 codes is one sequence's only visible key and value: the output is the value itself, exactly (with
    a scale of 1 all of them are bf16 numbers), the log-sum-exp its product with the query."""
    codes = torch.arange(256, dtype=torch.uint8, device=dev).view(F8)
    c = Case(dev, [0] * 256, T=T, Hq=Hq, Hkv=1, D=D, page=8, kv=F8, seed=1)
    c.scales = {"k_scale": torch.full((1,), 0.5, device=dev), "v_scale": torch.ones(1, device=dev)}
    c.kp.view(torch.uint8).zero_()
    for t in range(T):
        slot = c.table[:, t // 8].long()
        c.kp.view(torch.uint8)[slot, 0, t % 8, 3] = codes.view(torch.uint8)
        c.vp.view(torch.uint8)[slot, 0, t % 8] = codes.view(torch.uint8)[:, None]
    c.q = torch.zeros_like(c.q)
    c.q[..., 3] = 2
    o, lse = c.attend(scale=1.0, window=1)
    want = codes.float()
    assert want.isnan().sum() == 2
    ok = ~want.isnan()
    assert torch.equal(o.float()[ok], want[ok][:, None, None, None].expand(-1, T, Hq, D))
    assert o[~ok].isnan().all()
    # (the score goes to powers of two and back, and log2 of the sum, which is 1, is 0: three roundings)
    assert torch.allclose(lse[ok], want[ok][:, None, None].expand(-1, T, Hq), rtol=2.0 ** -21, atol=2.0 ** -21)
