"""The two ends of a language model over its vocabulary table: embed_take and its gradient, and
linear_softmax_loss and its gradient, against plain evaluations in 64 bits.

Tolerances are bounds of the arithmetic, derived per element before any run:
  u       half a unit in the last place of the result's type, relative (bf16 2^-8, fp16 2^-11, fp32 2^-24);
          fp16 results below its normal range are off by up to 2^-25 instead
  sums    k additions in binary32: k * 2^-23 relative to the sum of the magnitudes
          (2^-23, not 2^-24: the tensor cores may cut off where a rounding would round)
"""
import ctypes as C

import numpy as np
import pytest
import torch

import mshadow_b200
from mshadow_b200 import capi

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
U = {F16: 2.0 ** -11, BF16: 2.0 ** -8, F32: 2.0 ** -24}
TINY = {F16: 2.0 ** -25, BF16: 2.0 ** -134, F32: 2.0 ** -150}
ADD = 2.0 ** -23


@pytest.fixture(scope="module")
def lib():
    lb = mshadow_b200.load()
    if torch.cuda.is_available():
        lb.init(0)
    return lb


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def pitched(rows, cols, dtype, pad, offset=0, fill=None):
    """A rows x cols matrix with a row pitch of cols + pad, `offset` elements into its memory, and that memory."""
    base = torch.empty(offset + rows * (cols + pad) + 16, dtype=dtype, device="cuda")
    base.fill_(7.0 if fill is None else fill)
    return base[offset:offset + rows * (cols + pad)].view(rows, cols + pad)[:, :cols], base


def within(got, want, bound, what):
    got = got.double()
    assert torch.isfinite(got).all(), "%s: not finite" % what
    excess = (got - want).abs() - bound
    worst = excess.max().item() if excess.numel() else -1.0
    assert worst <= 0, "%s: beyond its bound by %g at %s" % (what, worst, torch.nonzero(excess == excess.max())[0].tolist())


# ---- refusals: answered on the host, so they are tested without a GPU ------------------------------------

def test_embed_refusals(lib):
    p = C.c_void_p(1 << 20)  # never dereferenced

    def take(n=4, rows=10, width=8, ld_dst=8, ld_table=8, dtype=0, dst=p, table=p, index=p):
        return lib.status("msb_embed_take", dst, table, index, n, rows, width, ld_dst, ld_table, dtype, 1.0, None)[0]

    assert take(dtype=1) == 1 and take(dtype=7) == 1
    assert take(n=-1) == 2 and take(rows=1 << 31) == 2 and take(width=-8) == 2
    assert take(ld_dst=7) == 2 and take(ld_table=4) == 2
    assert take(dst=None) == 1 and take(table=None) == 1 and take(index=None) == 1
    assert take(n=0, dst=None, table=None, index=None) == 0
    odd, two = C.c_void_p((1 << 20) + 1), C.c_void_p((1 << 20) + 2)
    assert take(dst=two) == 3 and take(table=two) == 3 and take(index=two) == 3 and take(dtype=2, dst=odd) == 3

    def grad(n=4, rows=10, width=8, ld_dst=8, ld_src=8, dtype=0, saver=0, dst=p, src=p, index=p, ws=None, size=0):
        return lib.status("msb_embed_take_grad", dst, src, index, n, rows, width, ld_dst, ld_src, dtype, 1.0, saver, ws,
                          size, None)[0]

    assert grad(dtype=3) == 1 and grad(saver=2) == 1
    assert grad(n=-1) == 2 and grad(ld_dst=7) == 2 and grad(ld_src=7) == 2
    assert grad(dst=None) == 1 and grad(src=None) == 1 and grad(index=None) == 1
    assert grad(n=100000, ws=p, size=1000) == 1  # workspace too small
    assert grad(dst=two) == 3 and grad(src=two) == 3 and grad(index=two) == 3
    assert grad(rows=0, dst=None, src=None, index=None) == 0
    assert grad(n=0, saver=1, dst=None, src=None, index=None) == 0
    assert lib.embed_take_grad_workspace(0, 64, 8) == 0
    assert lib.embed_take_grad_workspace(100000, 64, 8) > 0
    assert lib.status("msb_embed_take_grad_workspace", 4, 8, None)[0] == 1


def test_loss_refusals(lib):
    p = C.c_void_p(1 << 20)

    def loss(n=4, v=10, h=8, ld_x=8, ld_w=8, dtype=2, smooth=0.0, out=p, lse=p, x=p, w=p, label=p):
        return lib.status("msb_linear_softmax_loss", out, lse, x, w, label, n, v, h, ld_x, ld_w, dtype, -1, smooth, None, 0,
                          None)[0]

    assert loss(dtype=0) == 1 and loss(dtype=1) == 1
    assert loss(n=-1) == 2 and loss(v=0) == 2 and loss(h=0) == 2 and loss(v=1 << 31) == 2
    assert loss(ld_x=7) == 2 and loss(ld_w=7) == 2
    assert loss(smooth=-0.1) == 1 and loss(smooth=1.0) == 1 and loss(smooth=float("nan")) == 1
    assert loss(v=1, smooth=0.1) == 1
    for name in ("out", "lse", "x", "w", "label"):
        assert loss(**{name: None}) == 1
    assert loss(x=C.c_void_p((1 << 20) + 1)) == 3
    assert loss(n=0, out=None, lse=None, x=None, w=None, label=None) == 0

    def grad(n=4, v=10, h=8, ld=8, dtype=2, gw_dtype=2, saver=0, smooth=0.0, gx=p, gw=p, x=p, w=p, label=p, lse=p,
             ld_gw=8):
        return lib.status("msb_linear_softmax_loss_grad", gx, gw, x, w, label, lse, None, 1.0, n, v, h, ld, ld_gw, ld, ld,
                          dtype, gw_dtype, saver, -1, smooth, None, 0, None)[0]

    assert grad(dtype=0, gw_dtype=0) == 1 and grad(gw_dtype=12) == 1 and grad(dtype=12) == 1
    assert grad(saver=2) == 1 and grad(smooth=2.0) == 1
    assert grad(v=0) == 2 and grad(h=0) == 2 and grad(ld=7) == 2 and grad(ld_gw=7) == 2
    for name in ("x", "w", "label", "lse"):
        assert grad(**{name: None}) == 1
    assert grad(gw_dtype=0, gw=C.c_void_p((1 << 20) + 2)) == 3
    odd = C.c_void_p((1 << 20) + 2)  # 2-byte aligned: not an int32 or a float
    assert grad(label=odd) == 3 and grad(lse=odd) == 3
    for name in ("out", "lse", "label"):
        assert loss(**{name: odd}) == 3
    assert grad(gx=None, gw=None) == 0


def test_wrapper_refusals(lib):
    x = torch.zeros(4, 8, dtype=F16)
    w = torch.zeros(10, 8, dtype=F16)
    i = torch.zeros(4, dtype=torch.int32)
    f = torch.zeros(4)
    with pytest.raises(capi.MsbError):
        lib.embed_take(x, w.to(BF16), i)
    with pytest.raises(capi.MsbError):
        lib.embed_take(x, w, i.long())
    with pytest.raises(capi.MsbError):
        lib.embed_take(x, w, i[:3])
    with pytest.raises(capi.MsbError):
        lib.embed_take(x.double(), w.double(), i)
    with pytest.raises(capi.MsbError):
        lib.embed_take(x[:1].expand(4, 8), w, i)  # rows of the output overlap
    with pytest.raises(capi.MsbError):
        lib.embed_take(x, torch.zeros(8, 10, dtype=F16).t(), i)
    with pytest.raises(capi.MsbError):
        lib.embed_take_grad(w, x, torch.zeros(8, dtype=torch.int32)[::2])
    with pytest.raises(capi.MsbError):
        lib.linear_softmax_loss(f, f, x, w.to(BF16), i)
    with pytest.raises(capi.MsbError):
        lib.linear_softmax_loss(f, f[:2], x, w, i)
    with pytest.raises(capi.MsbError):
        lib.linear_softmax_loss(f.double(), f, x, w, i)
    with pytest.raises(capi.MsbError):
        lib.linear_softmax_loss_grad(x, w[:5], x, w, i, f)


# ---- look-up --------------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n,rows,width,pad,offset", [
    (1, 7, 1, 0, 0), (1, 500, 4096, 0, 0), (3, 1, 8, 0, 0), (17, 100, 33, 0, 0), (64, 50, 64, 8, 0), (64, 50, 64, 3, 0),
    (100, 300, 1001, 0, 0), (257, 64, 200, 0, 1), (1000, 333, 72, 0, 8), (5000, 40, 16, 0, 0), (4100, 999, 513, 5, 3)])
def test_embed_take(lib, dtype, n, rows, width, pad, offset):
    g = gen(n + rows + width)
    table, _ = pitched(rows, width, dtype, pad, offset)
    table.copy_(torch.randn(rows, width, device="cuda", generator=g))
    index = torch.randint(-2, rows + 3, (n,), device="cuda", generator=g).to(torch.int32)
    index[0] = rows - 1
    out, base = pitched(n, width, dtype, pad, offset)
    before = base.clone()
    for scale in (1.0, 0.37, -64.0):
        lib.embed_take(out, table, index, scale=scale)
        torch.cuda.synchronize()
        named = (index >= 0) & (index < rows)
        want = table[torch.where(named, index, 0).long()].double() * float(np.float32(scale)) * named[:, None]
        within(out, want, U[dtype] * want.abs() + TINY[dtype], "take")
        if scale == 1.0:
            assert torch.equal(out.double(), want)
        # memory around the rows stays as it was
        mask = torch.ones_like(base, dtype=torch.bool)
        mask[offset:offset + n * (width + pad)].view(n, width + pad)[:, :width] = False
        assert torch.equal(base[mask], before[mask])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("width", [1, 2, 3, 9, 31, 65, 127, 257, 511, 512, 513, 1025, 1537])
@pytest.mark.parametrize("at_table,at_out", [(0, 1), (1, 0), (1, 1)])
def test_embed_take_rows_anywhere(lib, dtype, width, at_table, at_out):
    """Around the segments and words that rows are cut into, the two sides starting at different parities."""
    g = gen(width + 2 * at_table + at_out)
    n, rows = 301, 67
    table, _ = pitched(rows, width, dtype, 0, at_table)
    table.copy_(torch.randn(rows, width, device="cuda", generator=g))
    index = torch.randint(-2, rows + 3, (n,), device="cuda", generator=g).to(torch.int32)
    out, base = pitched(n, width, dtype, at_out, at_out)
    before = base.clone()
    lib.embed_take(out, table, index, scale=-2.0)
    named = (index >= 0) & (index < rows)
    want = table[torch.where(named, index, 0).long()].double() * -2.0 * named[:, None]
    assert torch.equal(out.double(), want)
    out.copy_(torch.full_like(out, 7.0))
    assert torch.equal(base, before)


@pytest.mark.gpu
def test_embed_take_special_values(lib):
    """Infinities and NaN in rows that no index names reach nothing; in named rows they come out."""
    table = torch.randn(6, 40, device="cuda").to(BF16)
    table[1] = float("nan")
    table[2] = float("inf")
    index = torch.tensor([0, -1, 5, 6, 3, 1 << 30, -(1 << 31)], dtype=torch.int32, device="cuda")
    out = torch.full((7, 40), 3.0, dtype=BF16, device="cuda")
    lib.embed_take(out, table, index)
    assert torch.equal(out[[0, 2, 4]], table[[0, 5, 3]]) and (out[[1, 3, 5, 6]] == 0).all()
    lib.embed_take(out, table, torch.tensor([1, 2, 1, 2, 0, 0, 0], dtype=torch.int32, device="cuda"))
    assert out[[0, 2]].isnan().all() and (out[[1, 3]] == float("inf")).all() and torch.equal(out[4], table[0])
    lib.embed_take(out, table[:0], index)  # an empty table: no index names a row
    assert (out == 0).all()


# ---- gradient of the look-up ------------------------------------------------------------------------------------

def grad_oracle(dst, src, index, scale, add):
    rows = dst.shape[0]
    named = (index >= 0) & (index < rows)
    at = torch.where(named, index, 0).long()
    s = float(np.float32(scale))
    val = src.double() * named[:, None]
    total = torch.zeros(rows, src.shape[1], dtype=torch.float64, device="cuda").index_add_(0, at, val)
    mags = torch.zeros_like(total).index_add_(0, at, val.abs())
    count = torch.zeros(rows, dtype=torch.float64, device="cuda").index_add_(0, at, named.double())
    base = dst.double() if add else torch.zeros_like(total)
    want = base + s * total
    # count additions, the product with scale, and (adding) one more addition, all in binary32
    bound = ((count[:, None] + 2) * ADD) * abs(s) * mags + (ADD * want.abs() if add else 0)
    return want, bound + U[dst.dtype] * (want.abs() + bound) + TINY[dst.dtype]


def zipf(n, rows, g):
    mass = torch.arange(1, rows + 1, device="cuda", dtype=torch.float64).pow_(-1.1).cumsum_(0)
    return torch.searchsorted(mass, torch.rand(n, device="cuda", dtype=torch.float64, generator=g) * mass[-1]).clamp_(max=rows - 1).to(torch.int32)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("add", [False, True])
@pytest.mark.parametrize("n,rows,width,pad,offset,kind", [
    (1, 9, 5, 0, 0, "any"), (1, 300, 256, 0, 0, "any"), (31, 4, 16, 0, 0, "any"), (64, 1000, 1024, 0, 0, "any"),
    (512, 130, 200, 0, 0, "any"), (513, 130, 200, 0, 0, "any"), (512, 3, 40, 8, 0, "same"), (600, 2, 24, 0, 0, "same"),
    (64 * 20, 50, 64, 0, 0, "same"), (64 * 9 + 1, 700, 33, 0, 0, "any"), (4096, 5000, 72, 0, 0, "zipf"),
    (5003, 257, 513, 3, 1, "zipf"), (3000, 1, 129, 0, 0, "same"), (20000, 300, 40, 0, 0, "zipf"),
    (1000, 400, 65, 0, 0, "outside"), (100, 400, 64, 0, 0, "outside"), (4096, 64, 8, 0, 0, "runs")])
def test_embed_take_grad(lib, dtype, add, n, rows, width, pad, offset, kind):
    g = gen(n + 3 * rows + width)
    src, _ = pitched(n, width, dtype, pad, offset)
    src.copy_(torch.randn(n, width, device="cuda", generator=g))
    if kind == "any":
        index = torch.randint(0, rows, (n,), device="cuda", generator=g).to(torch.int32)
        index[n // 2] = -5 if n > 1 else rows - 1
    elif kind == "same":
        index = torch.full((n,), rows - 1, dtype=torch.int32, device="cuda")
    elif kind == "zipf":
        index = zipf(n, rows, g)
        index[::7] = rows + 2
    elif kind == "outside":
        index = torch.randint(rows, rows + 9, (n,), device="cuda", generator=g).to(torch.int32) * torch.tensor([1, -1], device="cuda", dtype=torch.int32).repeat(n // 2)
    else:  # runs of exactly 64: the longest that are not split, at every place of a chunk
        index = (torch.arange(n, device="cuda") // 64 % rows).to(torch.int32)
        index[5] = 0
    dst, base = pitched(rows, width, dtype, pad, offset)
    dst.copy_(torch.randn(rows, width, device="cuda", generator=g))
    dst[rows // 2] = -0.0
    before, start = base.clone(), dst.clone()
    for scale in (1.0, -2.5):
        dst.copy_(start)
        want, bound = grad_oracle(dst, src, index, scale, add)
        lib.embed_take_grad(dst, src, index, scale=scale, saver=int(add))
        torch.cuda.synchronize()
        within(dst, want, bound, "take_grad")
        again = torch.empty_like(start).copy_(start)
        lib.embed_take_grad(again, src, index, scale=scale, saver=int(add))
        assert torch.equal(again, dst), "equal calls differ"
        named = torch.zeros(rows, dtype=torch.bool, device="cuda")
        named[index[(index >= 0) & (index < rows)].long()] = True
        left = dst[~named]
        assert torch.equal(left, start[~named]) if add else (left == 0).all()
        mask = torch.ones_like(base, dtype=torch.bool)
        mask[offset:offset + rows * (width + pad)].view(rows, width + pad)[:, :width] = False
        assert torch.equal(base[mask], before[mask])


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1023, 1025, 16383, 16384, 16385])
@pytest.mark.parametrize("rows", [2, 500, 70000, 1500000])
def test_embed_take_grad_list_lengths(lib, n, rows):
    """Around the lengths where the way of sorting changes, with one to three digits per row number."""
    g = gen(n + rows)
    src = torch.randn(n, 8, device="cuda", generator=g)
    index = zipf(n, rows, g)
    index = torch.randperm(rows, device="cuda", generator=g).to(torch.int32)[index.long()]
    index[::11] = -1
    index[5::13] = rows
    dst = torch.empty(rows, 8, device="cuda")
    want, bound = grad_oracle(dst, src, index, 1.0, False)
    lib.embed_take_grad(dst, src, index)
    within(dst, want, bound, "take_grad")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_embed_take_grad_no_indices(lib, dtype):
    dst = torch.ones(300, 24, dtype=dtype, device="cuda")
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    src = torch.zeros(0, 24, dtype=dtype, device="cuda")
    lib.embed_take_grad(dst, src, none, saver=1)
    assert (dst == 1).all()
    lib.embed_take_grad(dst, src, none)
    assert (dst == 0).all()


@pytest.mark.gpu
def test_embed_take_grad_skipped_rows_may_hold_anything(lib):
    for n in (100, 3000):
        src = torch.randn(n, 64, device="cuda").to(F16)
        index = torch.randint(0, 50, (n,), device="cuda").to(torch.int32)
        index[::3] = -1
        index[1::6] = 50
        clean = src.clone()
        clean[(index < 0) | (index >= 50)] = 0
        src[::3] = float("nan")
        src[1::6] = float("inf")
        a, b = torch.empty(50, 64, dtype=F16, device="cuda"), torch.empty(50, 64, dtype=F16, device="cuda")
        lib.embed_take_grad(a, src, index)
        lib.embed_take_grad(b, clean, index)
        assert torch.equal(a, b) and torch.isfinite(a).all()


@pytest.mark.gpu
def test_embed_take_grad_against_differences(lib):
    """The gradient of sum(c * take(T)) with respect to T, from differences: the look-up is linear in T."""
    g = gen(3)
    table = torch.randn(40, 24, device="cuda", generator=g)
    index = torch.randint(0, 40, (700,), device="cuda", generator=g).to(torch.int32)
    c = torch.randn(700, 24, device="cuda", generator=g)
    grad = lib.embed_take_grad(torch.empty_like(table), c, index, scale=0.5)
    out = torch.empty_like(c)
    for r, k in ((0, 0), (7, 23), (39, 11), (20, 5)):
        def value(step):
            t = table.clone()
            t[r, k] = step  # exact values, so the products with 0.5 are exact too
            return (lib.embed_take(out, t, index, scale=0.5).double() * c.double()).sum().item()
        want = (value(2.0) - value(-2.0)) / 4.0
        mag = c[index == r, k].double().abs().sum().item()
        assert abs(grad[r, k].item() - want) <= 702 * ADD * 0.5 * mag + 1e-9 * c.double().abs().sum().item()


# ---- loss ---------------------------------------------------------------------------------------------------------

def problem(n, v, h, dtype, seed, pad_x=0, pad_w=0, off_x=0, off_w=0, ignored=0.0, spread=2.0):
    g = gen(seed)
    x, _ = pitched(n, h, dtype, pad_x, off_x)
    w, _ = pitched(v, h, dtype, pad_w, off_w)
    w.copy_(torch.randn(v, h, device="cuda", generator=g) * (spread / h ** 0.5))
    label = torch.randint(0, v, (n,), device="cuda", generator=g).to(torch.int32)
    x.copy_(torch.randn(n, h, device="cuda", generator=g) + w[label.long()].float())
    if ignored:
        label[torch.rand(n, device="cuda", generator=g) < ignored] = -1
    return x, w, label


def loss_oracle(x, w, label, ignore, smooth):
    """loss, lse, bounds, and what the gradient's oracle needs; 64 bits."""
    v, h = w.shape
    live = (label != ignore) & (label >= 0) & (label < v)
    xd = torch.where(live[:, None], x.double(), 0.0)
    wd = w.double()
    z = xd @ wd.t()
    dz = (h + 8) * ADD * (xd.abs() @ wd.abs().t()).amax(1)  # error of any logit of the row
    lse = torch.logsumexp(z, 1)
    at = torch.where(live, label, 0).long()[:, None]
    zl = z.gather(1, at)[:, 0]
    a = float(np.float32(smooth))
    rest = z.sum(1) - zl
    loss = lse - (1 - a) * zl - (a / (v - 1) * rest if a else 0.0)
    # the sum of exponentials: 8 additions per lane of a group, 3 joining, one group and one tile after another (a
    # tile in eight per thread); each exponential 2^-21; one rounding of the result
    tiles = -(-v // 256)
    rel = (8 + 3 + 2 * 8 + 2 * (tiles / 8 + 9)) * ADD + 2.0 ** -20
    e_lse = dz + rel + 2 * ADD * lse.abs()
    e_loss = e_lse + dz + ADD * (loss.abs() + lse.abs() + zl.abs())
    if a:
        e_loss = e_loss + a * (dz + (256 / 8 + tiles + 8) * ADD * z.abs().sum(1) / (v - 1))
    zero = torch.zeros_like(loss)
    return (torch.where(live, loss, zero), torch.where(live, lse, zero), torch.where(live, e_loss, zero),
            torch.where(live, e_lse, zero), dict(live=live, z=z, dz=dz, lse=lse, e_lse=e_lse, at=at, xd=xd, wd=wd, a=a))


def grad_bounds(q, gloss, scale, dtype, gw_dtype, base=None):
    live, z, wd, xd, a = q["live"], q["z"], q["wd"], q["xd"], q["a"]
    n, v = z.shape
    s = float(np.float32(scale)) * (torch.ones(n, dtype=torch.float64, device="cuda") if gloss is None else gloss.double())
    s = torch.where(live, s, torch.zeros_like(s))
    p = (z - q["lse"][:, None]).exp()
    t = torch.full_like(p, a / (v - 1) if a else 0.0)
    t.scatter_(1, q["at"], 1.0 - a)
    d = (p - t) * s[:, None]
    # d before its rounding: errors of z and lse (and of lse in base 2) in the exponent, the exponential, subtraction and product
    rho = q["dz"] + q["e_lse"] + 4 * ADD * (q["lse"].abs() + z.abs().amax(1)) + 2.0 ** -20
    e = (p * rho.expm1()[:, None] + 3 * ADD * (p + t)) * s.abs()[:, None]
    top = s.abs().max().item()
    e = e + U[dtype] * (d.abs() + e) + TINY[dtype] * (top * 2.0 ** -14 if top > 0 else 0.0)
    gx, gw = d @ wd, d.t() @ xd
    bx = e @ wd.abs() + (v + 16) * ADD * ((d.abs() + e) @ wd.abs())
    bw = e.t() @ xd.abs() + (n + 16) * ADD * ((d.abs() + e).t() @ xd.abs())
    if base is not None:
        gw = gw + base.double()
        bw = bw + ADD * gw.abs()
    return (gx, bx + U[dtype] * (gx.abs() + bx) + TINY[dtype], gw, bw + U[gw_dtype] * (gw.abs() + bw) + TINY[gw_dtype])


def check_loss(lib, x, w, label, ignore=-1, smooth=0.0):
    n = x.shape[0]
    loss, lse = torch.full((n,), 9.0, device="cuda"), torch.full((n,), 9.0, device="cuda")
    lib.linear_softmax_loss(loss, lse, x, w, label, ignore_label=ignore, smooth=smooth)
    torch.cuda.synchronize()
    lib.stream_wait(None)
    want, wlse, e_loss, e_lse, q = loss_oracle(x, w, label, ignore, smooth)
    within(lse, wlse, e_lse, "lse")
    within(loss, want, e_loss, "loss")
    again, lse2 = torch.empty_like(loss), torch.empty_like(lse)
    lib.linear_softmax_loss(again, lse2, x, w, label, ignore_label=ignore, smooth=smooth)
    assert torch.equal(again, loss) and torch.equal(lse2, lse), "equal calls differ"
    return loss, lse, q


SIZES = [(1, 1, 1), (1, 2, 8), (1, 1000, 64), (2, 257, 65), (5, 300, 7), (127, 255, 63), (128, 256, 64), (129, 257, 72),
         (130, 3000, 200), (256, 511, 128), (257, 513, 136), (300, 5003, 96), (511, 70, 520), (1000, 300, 33)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("n,v,h", SIZES)
def test_loss(lib, dtype, n, v, h):
    x, w, label = problem(n, v, h, dtype, n + v + h)
    check_loss(lib, x, w, label)


@pytest.mark.gpu
@pytest.mark.parametrize("n,v,h,smooth", [(1, 2, 16, 0.1), (40, 700, 64, 0.1), (300, 257, 100, 0.9), (3, 5000, 24, 0.25)])
def test_loss_smooth(lib, n, v, h, smooth):
    x, w, label = problem(n, v, h, BF16, n + v)
    check_loss(lib, x, w, label, smooth=smooth)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("pad_x,pad_w,off_x,off_w", [(8, 0, 0, 0), (3, 0, 0, 0), (0, 8, 8, 8), (0, 5, 1, 0), (0, 0, 0, 3), (1, 1, 1, 1)])
def test_loss_layouts(lib, dtype, pad_x, pad_w, off_x, off_w):
    for n, v, h in ((7, 600, 64), (300, 513, 72), (70, 400, 37)):
        x, w, label = problem(n, v, h, dtype, 5, pad_x, pad_w, off_x, off_w, ignored=0.2)
        check_loss(lib, x, w, label)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 60, 400, 1500])
def test_loss_rows_that_do_not_count(lib, n):
    x, w, label = problem(n, 700, 64, BF16, 11, ignored=0.5)
    label[n // 2] = 700
    label[n - 1] = -(1 << 31)
    label[0] = 5
    dead = (label < 0) | (label >= 700) | (label == 5)
    x[dead] = float("nan")
    x[dead & (torch.arange(n, device="cuda") % 2 == 0)] = float("inf")
    loss, lse, _ = check_loss(lib, x, w, label, ignore=5)
    assert (loss[dead] == 0).all() and (lse[dead] == 0).all()
    label.fill_(-100)
    loss, lse, _ = check_loss(lib, x, w, label)
    assert (loss == 0).all() and (lse == 0).all()


@pytest.mark.gpu
def test_loss_extreme_logits(lib):
    """Rows whose logits reach the thousands, equal logits, and one class far above the others."""
    x, w, label = problem(64, 900, 64, F16, 2, spread=300.0)
    x.mul_(4)
    check_loss(lib, x, w, label)
    x.zero_()
    loss, lse, _ = check_loss(lib, x, w, label)
    assert torch.allclose(lse, torch.full_like(lse, float(np.log(900))), rtol=2.0 ** -22)
    w.zero_()
    w[5, 0] = 200.0
    x[:, 0] = 4.0
    label.fill_(5)
    loss, _, _ = check_loss(lib, x, w, label)
    assert (loss == 0).all()


@pytest.mark.gpu
def test_loss_infinite_weights(lib):
    """A class at -infinity weighs nothing; a NaN or +infinity makes its row's loss NaN, and no other row's."""
    x, w, label = problem(40, 600, 64, BF16, 3)
    x[:, 0] = x[:, 0].abs() + 0.5
    w[300:] = 0
    w[300:, 0] = float("-inf")
    label.clamp_(max=299)
    loss, lse = torch.empty(40, device="cuda"), torch.empty(40, device="cuda")
    lib.linear_softmax_loss(loss, lse, x, w, label)
    want, wlse, e_loss, e_lse, _ = loss_oracle(x, w[:300], label, -1, 0.0)
    within(loss, want, e_loss, "loss beside classes at -infinity")
    x[7, 3] = float("nan")
    lib.linear_softmax_loss(loss, lse, x, w, label)
    others = torch.arange(40, device="cuda") != 7
    assert loss[7].isnan() and torch.isfinite(loss[others]).all()


@pytest.mark.gpu
def test_loss_long(lib):
    """Pieces: an unaligned table longer than the copy that is held of it, and many tiles of tokens."""
    x, w, label = problem(5, 70001, 1001, BF16, 1)
    check_loss(lib, x, w, label)
    x, w, label = problem(9000, 1000, 40, F16, 1, ignored=0.1)
    check_loss(lib, x, w, label)


# ---- gradient of the loss -----------------------------------------------------------------------------------------

def check_grad(lib, x, w, label, gloss=None, scale=1.0, ignore=-1, smooth=0.0, add=False, gw_dtype=None, pad=0, what="xw"):
    n, h = x.shape
    v = w.shape[0]
    gw_dtype = gw_dtype or x.dtype
    gx, bx_mem = pitched(n, h, x.dtype, pad)
    gw, bw_mem = pitched(v, h, gw_dtype, pad)
    start = None
    if add:
        gw.copy_(torch.randn(v, h, device="cuda", generator=gen(77)) * scale)
        start = gw.clone()
    keep_x, keep_w = bx_mem.clone(), bw_mem.clone()
    loss, lse = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    lib.linear_softmax_loss(loss, lse, x, w, label, ignore_label=ignore, smooth=smooth)

    def run():
        lib.linear_softmax_loss_grad(gx if "x" in what else None, gw if "w" in what else None, x, w, label, lse, gloss,
                                     scale, ignore_label=ignore, smooth=smooth, saver=int(add))
        torch.cuda.synchronize()
        lib.stream_wait(None)

    run()
    _, _, _, _, q = loss_oracle(x, w, label, ignore, smooth)
    wx, bx, ww, bw = grad_bounds(q, gloss, scale, x.dtype, gw_dtype, start)
    if "x" in what:
        within(gx, wx, bx, "gdata")
        assert (gx[~q["live"]] == 0).all()
    else:
        assert torch.equal(bx_mem, keep_x)
    if "w" in what:
        within(gw, ww, bw, "gweight")
    else:
        assert torch.equal(bw_mem, keep_w)
    if pad:  # memory between the rows stays as it was
        for mem, keep, rows in ((bx_mem, keep_x, n), (bw_mem, keep_w, v)):
            a = mem[:rows * (h + pad)].view(rows, h + pad)[:, h:]
            assert torch.equal(a, keep[:rows * (h + pad)].view(rows, h + pad)[:, h:])
            assert torch.equal(mem[rows * (h + pad):], keep[rows * (h + pad):])
    once = gx.clone(), gw.clone()
    if add:
        gw.copy_(start)
    run()
    assert torch.equal(gx, once[0]) and torch.equal(gw, once[1]), "equal calls differ"
    return gx, gw


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("n,v,h", SIZES)
def test_loss_grad(lib, dtype, n, v, h):
    x, w, label = problem(n, v, h, dtype, n + v + h, ignored=0.1 if n > 4 else 0.0)
    check_grad(lib, x, w, label, scale=1.0 / n)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("add", [False, True])
@pytest.mark.parametrize("pad", [0, 8, 3])
def test_loss_grad_outputs(lib, dtype, f32, add, pad):
    for n, v, h in ((60, 600, 64), (300, 300, 333)):
        x, w, label = problem(n, v, h, dtype, 9, ignored=0.3)
        gloss = torch.randn(n, device="cuda", generator=gen(4))
        gloss[::5] = 0.0
        check_grad(lib, x, w, label, gloss=gloss, scale=0.01, add=add, gw_dtype=F32 if f32 else None, pad=pad)


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["x", "w"])
def test_loss_grad_one_output(lib, what):
    x, w, label = problem(200, 700, 72, BF16, 9)
    check_grad(lib, x, w, label, what=what)


@pytest.mark.gpu
@pytest.mark.parametrize("n,v,h,smooth", [(1, 2, 16, 0.1), (140, 700, 64, 0.1), (300, 257, 100, 0.9)])
def test_loss_grad_smooth(lib, n, v, h, smooth):
    x, w, label = problem(n, v, h, F16, n + v, ignored=0.2 if n > 1 else 0.0)
    check_grad(lib, x, w, label, smooth=smooth, scale=1.0 / n)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.0, 1e-9, 1e-4, 3e5, -2.0])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_loss_grad_scales(lib, dtype, scale):
    """Small scales do not vanish in d and large ones do not overflow in it."""
    x, w, label = problem(150, 400, 64, dtype, 21)
    if dtype == F16 and scale > 1:
        x.mul_(2.0 ** -8)
        w.mul_(2.0 ** -8)
    gx, gw = check_grad(lib, x, w, label, scale=scale, gw_dtype=F32)
    assert (gw != 0).any() or scale == 0.0


@pytest.mark.gpu
@pytest.mark.parametrize("pad_x,pad_w,off_x,off_w", [(8, 0, 0, 0), (3, 5, 1, 1), (0, 0, 0, 3)])
def test_loss_grad_layouts(lib, pad_x, pad_w, off_x, off_w):
    for n, v, h in ((7, 600, 64), (300, 513, 37)):
        x, w, label = problem(n, v, h, BF16, 5, pad_x, pad_w, off_x, off_w, ignored=0.2)
        check_grad(lib, x, w, label, pad=1)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 60, 700])
def test_loss_grad_rows_that_do_not_count(lib, n):
    x, w, label = problem(n, 700, 64, BF16, 11, ignored=0.5)
    label[n // 2] = 700
    label[n - 1] = -(1 << 31)
    dead = (label < 0) | (label >= 700)
    x[dead] = float("nan")
    gloss = torch.ones(n, device="cuda")
    gloss[dead] = float("nan")
    check_grad(lib, x, w, label, gloss=gloss)
    label.fill_(-1)
    gx, gw = check_grad(lib, x, w, label, gloss=gloss)
    assert (gx == 0).all() and (gw == 0).all()
    check_grad(lib, x, w, label, gloss=gloss, add=True)


@pytest.mark.gpu
def test_loss_grad_no_tokens(lib):
    x = torch.zeros(0, 40, dtype=BF16, device="cuda")
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    w = torch.randn(50, 40, device="cuda").to(BF16)
    gw = torch.ones_like(w)
    e = torch.zeros(0, device="cuda")
    lib.linear_softmax_loss(e, e, x, w, none)
    lib.linear_softmax_loss_grad(x, gw, x, w, none, e, saver=1)
    assert (gw == 1).all()
    lib.linear_softmax_loss_grad(x, gw, x, w, none, e)
    assert (gw == 0).all()


@pytest.mark.gpu
def test_loss_grad_pieces(lib):
    """A vocabulary of several pieces: tokens enough that a piece of d holds fewer classes than there are."""
    x, w, label = problem(65700, 4500, 40, BF16, 5, ignored=0.05)
    check_grad(lib, x, w, label, scale=1.0 / 65700, gw_dtype=F32)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,gw_dtype,add", [(BF16, None, False), (F16, F32, True), (BF16, F32, False)])
def test_loss_grad_long(lib, dtype, gw_dtype, add):
    """Contractions and tables long enough for the widest tiles, with ends that fill none of them."""
    x, w, label = problem(8130, 8003, 2500, dtype, 5, ignored=0.05)
    check_grad(lib, x, w, label, scale=1.0 / 8130, gw_dtype=gw_dtype, add=add)


@pytest.mark.gpu
def test_loss_grad_unaligned_pieces(lib):
    x, w, label = problem(300, 70001, 1001, BF16, 1)
    check_grad(lib, x, w, label, scale=1.0 / 300)


@pytest.mark.gpu
def test_loss_grad_against_differences(lib):
    """Central differences of the 64-bit loss along single weights and features."""
    x, w, label = problem(30, 90, 24, F16, 8, ignored=0.2)
    smooth, scale = 0.1, 0.5
    gx, gw = check_grad(lib, x, w, label, smooth=smooth, scale=scale, gw_dtype=F32)
    _, _, _, _, q = loss_oracle(x, w, label, -1, smooth)
    _, bx, _, bw = grad_bounds(q, None, scale, F16, F32)

    def value(xd, wd):
        z = xd @ wd.t()
        a = q["a"]
        zl = z.gather(1, q["at"])[:, 0]
        per = torch.logsumexp(z, 1) - (1 - a) * zl - a / 89 * (z.sum(1) - zl)
        return (per * q["live"]).sum().item() * scale

    step = 1e-4
    for r, k in ((0, 0), (3, 23), (29, 11), (17, 5)):
        for grad, bound, pos in ((gx, bx, 0), (gw, bw, 1)):
            ends = []
            for sign in (1, -1):
                mats = [q["xd"].clone(), q["wd"].clone()]
                mats[pos][r, k] += sign * step
                ends.append(value(*mats))
            diff = (ends[0] - ends[1]) / (2 * step)
            # third derivative over six times step^2 (a few units here), and the differences' own rounding
            assert abs(grad[r, k].item() - diff) <= bound[r, k].item() + 1e-6


# ---- the C++ headers ----------------------------------------------------------------------------------------------

def cxx_suite():
    import os
    return C.CDLL(os.path.join(os.path.dirname(os.path.abspath(__file__)), "cxx", "libmsb_vocab_suite.so"))


def test_bf16_rounding():
    """The host conversions of bf16_t against torch's, on every bit pattern, every tie, and beyond the range."""
    bits = np.arange(1 << 16, dtype=np.uint32) << 16
    near = np.concatenate([bits, bits | 0x8000, bits | 0x7fff, bits | 0x8001]).view(np.float32)
    got, back = np.empty(near.size, np.uint16), np.empty(near.size, np.float32)
    vp = lambda a: a.ctypes.data_as(C.c_void_p)  # noqa: E731
    assert cxx_suite().msb_bf16_round(vp(near), vp(got), vp(back), near.size) == capi.BFLOAT16
    want = torch.from_numpy(near).to(torch.bfloat16)
    nan = np.isnan(near)
    assert np.isnan(back[nan]).all()
    assert np.array_equal(got[~nan].view(np.int16), want.view(torch.int16).numpy()[~nan])
    assert np.array_equal(back[~nan], want.float().numpy()[~nan])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_cxx_headers(lib, dtype):
    """The same step through Tensor handles and through the C entries: the same bits."""
    n, v, h = 333, 700, 72
    table, tokens, label, gtable, bufs, ws = tied(lib, n, v, h, dtype, 9)
    model_step(lib, table, tokens, label, gtable, bufs, ws, None)
    torch.cuda.synchronize()
    want = gtable.clone(), bufs[2].clone()
    gtable.fill_(1)
    bufs[2].fill_(1)
    fn = getattr(cxx_suite(), "msb_vocab_step_" + ("f16" if dtype == F16 else "bf16"))
    fn.argtypes = [C.c_void_p] * 8 + [C.c_int] * 3 + [C.c_float]
    torch.cuda.synchronize()
    p = [t.data_ptr() for t in (table, tokens, label, gtable, bufs[0], bufs[1], bufs[2], bufs[3])]
    assert fn(*p, n, v, h, 1.0 / n) == 0
    assert torch.equal(gtable, want[0]) and torch.equal(bufs[2], want[1])


# ---- streams, graphs, workspaces ----------------------------------------------------------------------------------

def model_step(lib, table, tokens, label, gtable, bufs, workspace, stream):
    """Embedding, loss and both gradients into one table (tied weights)."""
    h, gh, loss, lse = bufs
    scale = 1.0 / tokens.shape[0]
    lib.embed_take(h, table, tokens, scale=2.0, stream=stream)
    lib.linear_softmax_loss(loss, lse, h, table, label, workspace=workspace, stream=stream)
    lib.linear_softmax_loss_grad(gh, gtable, h, table, label, lse, scale=scale, workspace=workspace, stream=stream)
    lib.embed_take_grad(gtable, gh, tokens, scale=2.0, saver=1, workspace=workspace, stream=stream)


def tied(lib, n, v, h, dtype, seed):
    g = gen(seed)
    table = (torch.randn(v, h, device="cuda", generator=g) * (2.0 / h ** 0.5)).to(dtype)
    tokens = zipf(n, v, g)
    label = torch.roll(tokens, -1).contiguous()
    label[-1] = -1
    tokens[n // 3] = -1
    bufs = (torch.empty(n, h, dtype=dtype, device="cuda"), torch.empty(n, h, dtype=dtype, device="cuda"),
            torch.empty(n, device="cuda"), torch.empty(n, device="cuda"))
    size = max(lib.linear_softmax_loss_workspace(n, v, h, gradient=True), lib.embed_take_grad_workspace(n, v, h), 1)
    return table, tokens, label, torch.empty(v, h, dtype=dtype, device="cuda"), bufs, torch.empty(size, dtype=torch.uint8, device="cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("n,v,h,dtype", [(700, 1500, 128, BF16), (90, 600, 72, F16)])
def test_tied_step(lib, n, v, h, dtype):
    """The four operators as a model uses them, against automatic differentiation in 64 bits."""
    table, tokens, label, gtable, bufs, ws = tied(lib, n, v, h, dtype, 1)
    model_step(lib, table, tokens, label, gtable, bufs, ws, None)
    torch.cuda.synchronize()
    t = table.double().requires_grad_()
    named = (tokens >= 0)[:, None]
    hid = 2.0 * t[tokens.clamp(min=0).long()] * named
    assert torch.equal(bufs[0].double(), hid.detach())  # a power of two: exact
    live = label >= 0
    logp = torch.log_softmax(hid[live] @ t.t(), 1)
    loss = -logp[torch.arange(int(live.sum()), device="cuda"), label[live].long()]
    (loss.sum() / n).backward()
    # both paths' bounds: the head's gradient, the hidden state's gradient carried through the look-up's, and the two
    # roundings of the shared gradient (after the head, after the look-up)
    _, _, _, _, q = loss_oracle(bufs[0], table, label, -1, 0.0)
    gx, bx, gw, bw = grad_bounds(q, None, 1.0 / n, dtype, dtype)
    carried = torch.zeros_like(gw).index_add_(0, tokens.clamp(min=0).long(), 2.0 * bx * named)
    mags = torch.zeros_like(gw).index_add_(0, tokens.clamp(min=0).long(), 2.0 * (gx.abs() + bx) * named)
    bound = bw + carried + (n + 4) * ADD * mags + 2 * U[dtype] * (t.grad.abs() + bw + carried) + 2 * TINY[dtype]
    within(gtable, t.grad, bound, "tied gradient")


@pytest.mark.gpu
def test_streams_and_scratch(lib):
    """Another stream, with the stream's own scratch memory, gives the same bits."""
    table, tokens, label, gtable, bufs, ws = tied(lib, 800, 1000, 64, BF16, 2)
    model_step(lib, table, tokens, label, gtable, bufs, ws, None)
    torch.cuda.synchronize()
    want, loss = gtable.clone(), bufs[2].clone()
    for _ in range(2):
        s = torch.cuda.Stream()
        gtable.fill_(5)
        s.wait_stream(torch.cuda.current_stream())
        model_step(lib, table, tokens, label, gtable, bufs, None, s.cuda_stream)
        s.synchronize()
        lib.stream_wait(s.cuda_stream)
        assert torch.equal(gtable, want) and torch.equal(bufs[2], loss)


@pytest.mark.gpu
def test_two_calls_at_once(lib):
    """Two streams at once, each with its own workspace."""
    a, b = tied(lib, 2000, 3000, 128, BF16, 3), tied(lib, 1500, 2500, 128, F16, 4)
    wants = []
    for q in (a, b):
        model_step(lib, *q, None)
        torch.cuda.synchronize()
        wants.append(q[3].clone())
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for q, s in zip((a, b), streams):
            s.wait_stream(torch.cuda.current_stream())
            model_step(lib, *q, s.cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(a[3], wants[0]) and torch.equal(b[3], wants[1])


@pytest.mark.gpu
def test_graph(lib):
    """Captured and replayed on new contents; a capture without a workspace is refused and leaves the capture usable."""
    q = tied(lib, 600, 900, 64, BF16, 5)
    table, tokens, label, gtable, bufs, ws = q
    model_step(lib, *q, None)  # the first call on a device precedes the capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s = torch.cuda.current_stream().cuda_stream
        with pytest.raises(capi.MsbError) as e:
            lib.linear_softmax_loss(bufs[2], bufs[3], bufs[0], table, label, stream=s)
        assert e.value.status == 1 and "graph" in str(e.value)
        with pytest.raises(capi.MsbError):
            lib.linear_softmax_loss_grad(bufs[1], gtable, bufs[0], table, label, bufs[3], stream=s)
        with pytest.raises(capi.MsbError):
            lib.embed_take_grad(gtable, bufs[1], tokens, stream=s)
        model_step(lib, *q, s)
    for seed in (6, 7):
        other = tied(lib, 600, 900, 64, BF16, seed)
        model_step(lib, *other, None)
        table.copy_(other[0])
        tokens.copy_(other[1])
        label.copy_(other[2])
        gtable.fill_(3)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(gtable, other[3]) and torch.equal(bufs[2], other[4][2])


@pytest.mark.gpu
def test_workspace_too_small(lib):
    x, w, label = problem(300, 700, 64, BF16, 1)
    f = torch.zeros(300, device="cuda")
    small = torch.empty(1000, dtype=torch.uint8, device="cuda")
    with pytest.raises(capi.MsbError):
        lib.linear_softmax_loss(f, f.clone(), x, w, label, workspace=small)
    with pytest.raises(capi.MsbError):
        lib.linear_softmax_loss_grad(None, torch.empty_like(w), x, w, label, f, workspace=small)
    # an odd address inside a large enough workspace serves
    size = lib.linear_softmax_loss_workspace(300, 700, 64)
    ws = torch.empty(size + 1, dtype=torch.uint8, device="cuda")[1:]
    loss, lse = torch.empty(300, device="cuda"), torch.empty(300, device="cuda")
    lib.linear_softmax_loss(loss, lse, x, w, label, workspace=ws)
    want, wlse, e_loss, e_lse, _ = loss_oracle(x, w, label, -1, 0.0)
    within(loss, want, e_loss, "loss")


@pytest.mark.gpu
def test_host_memory_is_refused(lib):
    """Pointers that a kernel could not follow are answered with an error, not with a fault."""
    d = lambda *shape: torch.zeros(*shape, dtype=BF16, device="cuda")  # noqa: E731
    i = torch.zeros(4, dtype=torch.int32, device="cuda")
    f = torch.zeros(4, device="cuda")
    bad = [lambda: lib.embed_take(d(4, 8), torch.zeros(9, 8, dtype=BF16), i),
           lambda: lib.embed_take(d(4, 8), d(9, 8), i.cpu()),
           lambda: lib.embed_take(d(4, 8), torch.zeros(9, 8, dtype=BF16).pin_memory(), i),
           lambda: lib.embed_take_grad(d(9, 8), torch.zeros(4, 8, dtype=BF16), i),
           lambda: lib.linear_softmax_loss(f, f.clone(), d(4, 8), torch.zeros(9, 8, dtype=BF16), i),
           lambda: lib.linear_softmax_loss(f, f.cpu(), d(4, 8), d(9, 8), i),
           lambda: lib.linear_softmax_loss(f, f.clone(), d(4, 8), d(9, 8), i, workspace=torch.empty(1 << 20, dtype=torch.uint8)),
           lambda: lib.linear_softmax_loss_grad(d(4, 8), torch.zeros(9, 8, dtype=BF16), d(4, 8), d(9, 8), i, f)]
    for call in bad:
        with pytest.raises(capi.MsbError) as e:
            call()
        assert e.value.status == 1
    lib.embed_take(d(4, 8), d(9, 8), i)
    torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("n", [16300, 16500, 70000])
def test_loss_long_token_lists(lib, n):
    """Around the length from which the live tokens are counted by a kernel of their own."""
    x, w, label = problem(n, 300, 24, BF16, 3, ignored=0.4)
    gloss = torch.randn(n, device="cuda", generator=gen(1))
    gloss[label < 0] = float("inf")
    check_loss(lib, x, w, label)
    check_grad(lib, x, w, label, gloss=gloss, scale=1e-3)


@pytest.mark.gpu
def test_gradient_in_place(lib):
    """gdata may be data itself: its rows are written after everything has been read."""
    for n in (40, 700):
        x, w, label = problem(n, 900, 64, BF16, 13, ignored=0.1)
        loss, lse = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
        lib.linear_softmax_loss(loss, lse, x, w, label)
        gx, gw, gw2 = torch.empty_like(x), torch.empty_like(w), torch.empty_like(w)
        lib.linear_softmax_loss_grad(gx, gw, x, w, label, lse)
        lib.linear_softmax_loss_grad(x, gw2, x, w, label, lse)
        assert torch.equal(x, gx) and torch.equal(gw, gw2)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [100, 3000])
@pytest.mark.parametrize("scale", [-2.0, float("inf"), float("nan")])
def test_dropped_indices_touch_no_row(lib, n, scale):
    """Indices that name no row leave every row's bits alone, whatever the scale (they are sorted among those of row 0)."""
    index = torch.full((n,), -1, dtype=torch.int32, device="cuda")
    index[1::2] = 50
    src = torch.randn(n, 24, device="cuda")
    dst = torch.full((50, 24), -0.0, device="cuda")
    lib.embed_take_grad(dst, src, index, scale=scale, saver=1)
    assert (dst.view(torch.int32) == -(1 << 31)).all()
    lib.embed_take_grad(dst, src, index, scale=scale)
    assert (dst.view(torch.int32) == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("n,v,h", [(5, 300, 40), (300, 700, 72), (700, 3000, 520), (3000, 20000, 264)])
def test_what_the_workspace_held_does_not_matter(lib, n, v, h):
    """NaN everywhere in the workspace gives the same bits as zeros."""
    table, tokens, label, gtable, bufs, ws = tied(lib, n, v, h, BF16, 21)
    label[::3] = -1
    seen = []
    for fill in (0, 0xff):
        ws.fill_(fill)
        lib.embed_take(bufs[0], table, tokens)
        lib.linear_softmax_loss(bufs[2], bufs[3], bufs[0], table, label, smooth=0.1, workspace=ws)
        ws.fill_(fill)
        lib.linear_softmax_loss_grad(bufs[1], gtable, bufs[0], table, label, bufs[3], smooth=0.1, workspace=ws)
        ws.fill_(fill)
        head = gtable.clone()
        lib.embed_take_grad(gtable, bufs[1], tokens, saver=1, workspace=ws)
        seen.append([t.clone() for t in (*bufs, head, gtable)])
    assert all(torch.equal(a, b) for a, b in zip(*seen))
    assert all(torch.isfinite(t).all() for t in seen[0])


@pytest.mark.gpu
def test_graph_of_kernels_not_used_before(lib):
    """A capture may use sizes, and with them kernels, that no earlier call used; two graphs with a workspace each."""
    x, w, label = problem(3, 40, 8, F16, 1)
    lib.linear_softmax_loss(torch.empty(3, device="cuda"), torch.empty(3, device="cuda"), x, w, label)
    torch.cuda.synchronize()
    runs = []
    for n, v, h in ((900, 9000, 1304), (77, 1300, 24)):
        q = tied(lib, n, v, h, F16, n)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            model_step(lib, *q, torch.cuda.current_stream().cuda_stream)
        runs.append((q, graph))
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        for (q, graph), s in zip(runs, (a, b)):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for q, _ in runs:
        got = q[3].clone()
        model_step(lib, *q, None)
        torch.cuda.synchronize()
        assert torch.equal(got, q[3])


@pytest.mark.gpu
def test_offsets_beyond_32_bits(lib):
    """Tables and token matrices of more than 2^31 elements: rows at the far end."""
    v, h, n = 530000, 4104, 40
    g = gen(1)
    w = torch.empty(v, h, dtype=BF16, device="cuda")
    for at in range(0, v, 50000):
        w[at:at + 50000] = torch.randn(min(50000, v - at), h, device="cuda", generator=g) * (2.0 / h ** 0.5)
    index = torch.tensor([v - 1, 0, v - 2, v // 2] * (n // 4), dtype=torch.int32, device="cuda")
    x = torch.empty(n, h, dtype=BF16, device="cuda")
    lib.embed_take(x, w, index)
    assert torch.equal(x, w[index.long()])
    label = index.flip(0).contiguous()
    loss, lse = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    lib.linear_softmax_loss(loss, lse, x, w, label)
    z = torch.cat([x.double() @ w[at:at + 50000].double().t() for at in range(0, v, 50000)], 1)
    want = torch.logsumexp(z, 1)
    e_z = (h + 8) * ADD * max((x.abs().double() @ w[at:at + 50000].abs().double().t()).max().item() for at in range(0, v, 50000))
    assert ((lse.double() - want).abs() <= e_z + 2.0 ** -15 + 2 * ADD * want.abs()).all()
    gw, gx = torch.empty_like(w), torch.empty_like(x)
    lib.linear_softmax_loss_grad(gx, gw, x, w, label, lse, scale=1.0 / n)
    far = torch.arange(v - 5, v, device="cuda")
    d = (z[:, far] - want[:, None]).exp() - (label[:, None] == far[None]).double()
    ref = d.t() @ x.double() / n
    assert ((gw[far].double() - ref).abs() <= (U[BF16] * 4) * (d.abs().t() @ x.abs().double()) / n + 1e-7).all()
    lib.embed_take_grad(gw, gx, index)
    ref = torch.zeros(5, h, dtype=torch.float64, device="cuda")
    for i in range(n):
        if int(index[i]) >= v - 5:
            ref[int(index[i]) - (v - 5)] += gx[i].double()
    assert ((gw[far].double() - ref).abs() <= U[BF16] * 2 * ref.abs() + 1e-9).all()
    del w, gw, z
    torch.cuda.empty_cache()
    n, v, h = 530000, 48, 4104
    x = torch.empty(n, h, dtype=F16, device="cuda")
    for at in range(0, n, 50000):
        x[at:at + 50000] = torch.randn(min(50000, n - at), h, device="cuda", generator=g)
    w = (torch.randn(v, h, device="cuda", generator=g) * (2.0 / h ** 0.5)).to(F16)
    label = torch.randint(0, v, (n,), device="cuda", generator=g).to(torch.int32)
    label[7] = -1
    loss, lse = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    lib.linear_softmax_loss(loss, lse, x, w, label)
    gx = torch.empty_like(x)
    lib.linear_softmax_loss_grad(gx, None, x, w, label, lse)
    far = slice(n - 300, n)
    want, wlse, e_loss, e_lse, q = loss_oracle(x[far], w, label[far], -1, 0.0)
    within(loss[far], want, e_loss, "loss")
    wx, bx, _, _ = grad_bounds(q, None, 1.0, F16, F16)
    within(gx[far], wx, bx, "gdata")
    assert (gx[7] == 0).all()


# ---- values that are not finite, and calls that nothing reaches -----------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("n,ignored", [(1, 0.0), (40, 0.0), (64, 0.0), (100, 0.0), (257, 0.0), (300, 0.3), (700, 0.5)])
def test_loss_grad_infinite_weights(lib, dtype, n, ignored):
    """Classes at -infinity (a weight that acts as a mask) have no gradient, and the other classes have theirs."""
    x, w, label = problem(n, 600, 64, dtype, 3, ignored=ignored)
    x[:, 0] = x[:, 0].abs() + 0.5
    w[300:] = 0
    w[300:, 0] = float("-inf")
    label.clamp_(max=299)
    loss, lse = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    for gw_dtype in (dtype, F32):
        for lab in (label, torch.full_like(label, -1)):
            lib.linear_softmax_loss(loss, lse, x, w, lab)
            gw = torch.full((600, 64), 5.0, dtype=gw_dtype, device="cuda")
            lib.linear_softmax_loss_grad(None, gw, x, w, lab, lse, scale=1.0 / n)
            _, _, _, _, q = loss_oracle(x, w[:300], lab, -1, 0.0)
            _, _, want, bound = grad_bounds(q, None, 1.0 / n, dtype, gw_dtype)
            within(gw[:300], want, bound, "gweight beside classes at -infinity")
            assert (gw[300:] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [float("inf"), float("nan"), -1.0])
@pytest.mark.parametrize("n,h", [(40, 64), (700, 72), (300, 33)])
def test_loss_grad_of_nothing(lib, n, h, scale):
    """No token counts, and the scale is one over their number: empty sums are zero whatever they are scaled by."""
    x, w, label = problem(n, 500, h, BF16, 6)
    dead = torch.full_like(label, -1)
    loss, lse = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    lib.linear_softmax_loss(loss, lse, x, w, dead)
    for gw_dtype in (BF16, F32):
        gx, gw = torch.full_like(x, 5.0), torch.full((500, h), 5.0, dtype=gw_dtype, device="cuda")
        lib.linear_softmax_loss_grad(gx, gw, x, w, dead, lse, scale=scale)
        assert (gx == 0).all() and (gw == 0).all()
        gw.fill_(5.0)
        lib.linear_softmax_loss_grad(gx, gw, x, w, dead, lse, scale=scale, saver=1)
        assert (gx == 0).all() and (gw == 5).all()
    # beside tokens that count the others' rows are zero all the same
    dead[3] = label[3]
    lib.linear_softmax_loss(loss, lse, x, w, dead)
    lib.linear_softmax_loss_grad(gx, gw, x, w, dead, lse, scale=scale)
    others = torch.arange(n, device="cuda") != 3
    assert (gx[others] == 0).all() and bool(torch.isfinite(gx[3]).all()) == (scale == -1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,word,nan", [(F32, torch.int32, 0x7fc12345), (F32, torch.int32, -0x3edcbb), (F16, torch.int16, 0x7e41),
                                            (F16, torch.int16, -0x1bf), (BF16, torch.int16, 0x7fc1), (BF16, torch.int16, -0x3f)])
@pytest.mark.parametrize("n", [100, 600, 3000, 9000, 20000])
@pytest.mark.parametrize("width,at", [(24, 0), (33, 1), (300, 0)])
def test_rows_not_named_keep_their_bits(lib, dtype, word, nan, n, width, at):
    """Added gradients leave rows alone that no index names, NaN bits too: dropped indices in lists of every kind of
    sort, with few and with many entries, beside named rows and by themselves."""
    rows = 50
    src, _ = pitched(n, width, dtype, 0, at)
    src.copy_(torch.randn(n, width, device="cuda", generator=gen(n)))
    for named, dropped in ((0, n), (n // 2, n // 2), (n - 40, 40), (n - 130, 130), (n - 3, 3)):
        index = torch.randint(1, rows - 1, (n,), device="cuda", generator=gen(n)).to(torch.int32)
        index[named:named + dropped] = -1
        index[named + dropped // 3:named + dropped] = rows + 7
        dst, _ = pitched(rows, width, dtype, 0, at)
        bits = torch.full((rows, width), nan, dtype=word, device="cuda")
        dst.copy_(bits.view(dtype))  # copies keep bits
        assert torch.equal(dst.contiguous().view(word), bits)
        lib.embed_take_grad(dst, src, index, scale=0.5, saver=1)
        left = torch.ones(rows, dtype=torch.bool, device="cuda")
        left[index[(index >= 0) & (index < rows)].long()] = False
        assert left[0] and left[rows - 1]
        assert (dst.contiguous().view(word)[left] == nan).all() and dst[~left].isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("n", [600, 5000, 12000])
def test_two_streams_add_into_one_table(lib, n):
    """Two calls at once into the same table: the rows that they name are disjoint, and both lists hold dropped indices, which
    are sorted among those of the first and the last row."""
    rows, width = 40, 2048
    dst = torch.zeros(rows, width, device="cuda")
    halves = []
    for k in range(2):
        index = torch.randint(0, rows // 2, (n,), device="cuda", generator=gen(k)).to(torch.int32)
        if k:
            index += rows // 2  # the last row is named here, the first one there
        index[::5] = -1 - k
        index[1::5] = rows + k
        src = torch.randint(-4, 5, (n, width), device="cuda", generator=gen(9 + k)).float()  # sums are exact
        ws = torch.empty(lib.embed_take_grad_workspace(n, rows, width), dtype=torch.uint8, device="cuda")
        halves.append((src, index, ws, torch.cuda.Stream()))
    want = torch.zeros(rows, width, dtype=torch.float64, device="cuda")
    for src, index, _, _ in halves:
        named = (index >= 0) & (index < rows)
        want.index_add_(0, index[named].long(), src[named].double())
    torch.cuda.synchronize()
    calls = 30
    for _ in range(calls):
        for src, index, ws, s in halves:
            lib.embed_take_grad(dst, src, index, saver=1, workspace=ws, stream=s.cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(dst.double(), calls * want)


@pytest.mark.gpu
def test_small_workspace_is_an_argument(lib):
    """A workspace that is too small is answered with the same status by all entries, and the call does nothing."""
    x, w, label = problem(700, 900, 64, BF16, 1)
    loss, lse = torch.full((700,), 9.0, device="cuda"), torch.full((700,), 9.0, device="cuda")
    gx, gw = torch.full_like(x, 9.0), torch.full_like(w, 9.0)
    for size in (1, 1000):
        small = torch.empty(size, dtype=torch.uint8, device="cuda")
        for call in (lambda: lib.linear_softmax_loss(loss, lse, x, w, label, workspace=small),
                     lambda: lib.linear_softmax_loss_grad(gx, gw, x, w, label, lse, workspace=small),
                     lambda: lib.embed_take_grad(gw, x, label, workspace=small)):
            with pytest.raises(capi.MsbError) as e:
                call()
            assert e.value.status == 1 and "workspace" in str(e.value)
    torch.cuda.synchronize()
    assert all((t == 9).all() for t in (loss, lse, gx, gw))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [5121, 7169, 8191, 8192, 8193])
@pytest.mark.parametrize("rows", [2, 500, 70000, 1500000])
def test_embed_take_grad_where_one_cta_stops_sorting(lib, n, rows):
    """The longest lists that one CTA sorts, all its rounds and all its shared memory, and the first that it does not, with
    one to three digits per row number."""
    g = gen(n + rows)
    src = torch.randn(n, 8, device="cuda", generator=g)
    index = zipf(n, rows, g)
    index = torch.randperm(rows, device="cuda", generator=g).to(torch.int32)[index.long()]
    index[::11] = -1
    index[5::13] = rows
    for add in (False, True):
        dst = torch.randn(rows, 8, device="cuda", generator=g)
        want, bound = grad_oracle(dst, src, index, 1.0, add)
        lib.embed_take_grad(dst, src, index, saver=int(add))
        within(dst, want, bound, "take_grad")


def own_row_bounds(q, gloss, scale, dtype):
    """gdata of tokens that count and its bound as in grad_bounds, but with what d loses below binary16's normal range counted in
    the token's own |gloss|: its row of d is stored 2^8 times that / (1 - a) or larger, so half of the smallest
    binary16 number is at most 2^-33 of it."""
    s = float(np.float32(scale)) * gloss.double()
    p = (q["z"] - q["lse"][:, None]).exp()
    v = p.shape[1]
    t = torch.full_like(p, q["a"] / (v - 1) if q["a"] else 0.0)
    t.scatter_(1, q["at"], 1.0 - q["a"])
    d = (p - t) * s[:, None]
    rho = q["dz"] + q["e_lse"] + 4 * ADD * (q["lse"].abs() + q["z"].abs().amax(1)) + 2.0 ** -20
    e = (p * rho.expm1()[:, None] + 3 * ADD * (p + t)) * s.abs()[:, None]
    e = e + U[dtype] * (d.abs() + e) + TINY[dtype] * 2.0 ** -8 * s.abs()[:, None]
    gx = d @ q["wd"]
    bx = e @ q["wd"].abs() + (v + 16) * ADD * ((d.abs() + e) @ q["wd"].abs())
    return gx, bx + U[dtype] * (gx.abs() + bx) + TINY[dtype]


@pytest.mark.gpu
@pytest.mark.parametrize("n,v,h,smooth", [(60, 40000, 64, 0.0), (300, 9000, 72, 0.1), (17000, 600, 40, 0.0)])
@pytest.mark.parametrize("largest", [1.0, 4096.0, float("inf"), float("nan")])
def test_loss_grad_of_unlike_tokens(lib, n, v, h, smooth, largest):
    """Tokens whose gloss lie many binary16 ranges apart, over flat distributions: each token's gdata is as exact as if it were
    alone; an infinite gloss spoils its own token and the weight's gradient, no other token's."""
    x, w, label = problem(n, v, h, F16, 17, ignored=0.2, spread=0.25)
    x.mul_(0.25)
    gloss = torch.exp2(-24.0 * torch.rand(n, device="cuda", generator=gen(2)))
    gloss[::4] = -gloss[::4]
    gloss[1::9] = 0.0
    label[n // 2] = 1
    gloss[n // 2] = largest
    usual = torch.isfinite(gloss)
    loss, lse = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    lib.linear_softmax_loss(loss, lse, x, w, label, smooth=smooth)
    _, _, _, _, q = loss_oracle(x, w, label, -1, smooth)
    counts = (q["live"] & usual).nonzero()[:, 0]
    for scale in (1.0, 2.0 ** 12):  # the largest leave binary16's range then, the others must not care
        gx, gw = torch.full_like(x, 9.0), torch.full((v, h), 9.0, device="cuda")
        lib.linear_softmax_loss_grad(gx, gw, x, w, label, lse, gloss, scale, smooth=smooth)
        part = dict(q, **{k: q[k][counts] for k in ("z", "lse", "dz", "e_lse", "at")})
        want, bound = own_row_bounds(part, gloss[counts], scale, F16)
        inside = (want.abs() + bound).amax(1) < 60000
        assert inside.sum() >= counts.numel() // 2
        within(gx[counts][inside], want[inside], bound[inside], "gdata")
        assert (gx[~q["live"]] == 0).all()
        if np.isfinite(largest):
            _, _, ww, bw = grad_bounds(q, gloss, scale, F16, F32)
            within(gw, ww, bw, "gweight")
        only = torch.full_like(x, 9.0)  # without the weight's gradient: the same
        lib.linear_softmax_loss_grad(only, None, x, w, label, lse, gloss, scale, smooth=smooth)
        assert torch.equal(only.view(torch.int16), gx.view(torch.int16))
        alone = torch.empty_like(gw)
        lib.linear_softmax_loss_grad(None, alone, x, w, label, lse, gloss, scale, smooth=smooth)
        if np.isfinite(largest):
            within(alone, ww, bw, "gweight alone")


# ---- long sums: the tensor cores cut off each time they add, so what is added in one go is bounded --------------------

RUN = 512 * ADD  # a run of 8192 elements is 512 additions, each off by up to one unit in the last place of the sum; where the
#                  sum is rounded to 16 bits, runs are twice as long


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("n,v,h,gw_dtype,add", [
    (65536, 256, 64, F32, False), (262144, 256, 64, F32, False), (262144, 256, 64, None, False), (200001, 300, 33, F32, False),
    (200001, 300, 33, None, True), (150000, 256, 40, None, True), (120000, 256, 64, F32, True), (16500, 40000, 512, F32, False),
    (16500, 40000, 512, None, False)])
def test_weight_gradient_of_a_frequent_class(lib, dtype, n, v, h, gw_dtype, add):
    """Every token names one class and all its terms have one sign: what is lost in each addition adds up."""
    gw_dtype = gw_dtype or dtype
    x = (torch.rand(n, h, device="cuda", generator=gen(n)) + 1).to(dtype)
    w = torch.zeros(v, h, device="cuda", dtype=dtype)
    label = torch.full((n,), 3, dtype=torch.int32, device="cuda")
    loss, lse = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    lib.linear_softmax_loss(loss, lse, x, w, label)
    gw = torch.ones(v, h, dtype=gw_dtype, device="cuda")
    lib.linear_softmax_loss_grad(None, gw, x, w, label, lse, scale=1.0 / n, saver=int(add))
    mean = x.double().mean(0)
    for row, d in ((3, 1.0 / v - 1.0), (4, 1.0 / v)):
        sums = d * mean
        # d: the exponential and lse (2^-20), a rounding; the sum: a run, and the runs; scale and result
        off = (2.0 ** -20 * (1.0 / v if row == 4 else 1.0) / abs(d) + U[dtype] + RUN * (1 if gw_dtype == F32 else 2) + (n / 8192 + 8) * ADD) * sums.abs()
        if row == 3 and v == 256:
            off -= U[dtype] * sums.abs()  # 255 / 256 has eight bits
        want = sums + (1.0 if add else 0.0)
        bound = off + ADD * want.abs() + U[gw_dtype] * (want.abs() + off) + TINY[gw_dtype]
        within(gw[row], want, bound, "gweight of class %d" % row)


@pytest.mark.gpu
@pytest.mark.parametrize("n,v,h", [(8, 1 << 20, 1024), (600, 131072, 4096), (300, 200003, 72), (129, 100000, 520)])
def test_data_gradient_over_a_long_vocabulary(lib, n, v, h):
    """Behind the label's term, by far the largest, every class adds one of the other sign."""
    w = torch.empty(v, h, dtype=F16, device="cuda")
    for at in range(0, v, 1 << 17):
        w[at:at + (1 << 17)] = torch.rand(min(1 << 17, v - at), h, device="cuda", generator=gen(at)) + 1
    w[0] = 100
    x = torch.zeros(n, h, device="cuda", dtype=F16)
    label = torch.zeros(n, dtype=torch.int32, device="cuda")
    loss, lse, gx = torch.empty(n, device="cuda"), torch.empty(n, device="cuda"), torch.empty_like(x)
    lib.linear_softmax_loss(loss, lse, x, w, label)
    lib.linear_softmax_loss_grad(gx, None, x, w, label, lse)
    mean = torch.stack([w[at:at + (1 << 17)].double().sum(0) for at in range(0, v, 1 << 17)]).sum(0) / v
    want = mean - 100
    # d: 1 - 1 / v is rounded to 1, and 1 / v is rounded (and 2^-20 for the exponential); sums are up to 102 large
    off = 102 * (2 * RUN + (v / 8192 + 16) * ADD) + 100.0 / v + mean * (U[F16] + 2.0 ** -20)
    within(gx, want.expand(n, h), (off + U[F16] * (want.abs() + off)).expand(n, h), "gdata")


@pytest.mark.gpu
@pytest.mark.parametrize("n,v,h", [(64, 512, 65536), (300, 20000, 16384), (40, 300, 12345)])
def test_gradient_over_many_features(lib, n, v, h):
    """Logits whose terms have one sign: those of the gradient are as exact as lse needs them."""
    x = (torch.rand(n, h, device="cuda", generator=gen(h)) + 1).to(F16)
    w = torch.full((v, h), 20.0 / 1.5 / h, device="cuda", dtype=F16)
    label = torch.full((n,), 3, dtype=torch.int32, device="cuda")
    loss, lse = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    lib.linear_softmax_loss(loss, lse, x, w, label)
    gw = torch.empty(v, h, device="cuda")
    lib.linear_softmax_loss_grad(None, gw, x, w, label, lse, scale=1.0 / n)
    z = (x.double() @ w[0].double()).max().item()
    # all logits of a token are equal: p = 1 / v, off by what the two logits are (in runs of 8192 features, 512 additions)
    rho = z * (512 + 64 + h / 8192 + h / 1024 + 16) * ADD + 2.0 ** -19
    want = x.double().mean(0) / v
    rows = torch.arange(v, device="cuda") != 3
    within(gw[rows], want.expand(v - 1, h), (want * (rho + U[F16] + (n + 16) * ADD)).expand(v - 1, h), "gweight")


def test_headers_without_the_operators(tmp_path):
    """A program that includes the headers and calls none of these operators builds for architectures without tcgen05."""
    import os
    import shutil
    import subprocess
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("nvcc not found")
    src = tmp_path / "user.cu"
    src.write_text("#include <mshadow/tensor.h>\nint rows(mshadow::Tensor<mshadow::gpu, 2, float> t) { return t.size(0); }\n")
    inc = os.path.join(os.path.dirname(os.path.abspath(mshadow_b200.__file__)), "include")
    done = subprocess.run([nvcc, "-std=c++11", "-arch=sm_100", "-I" + inc, "-cubin", str(src), "-o", str(tmp_path / "user.cubin")],
                          capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


@pytest.mark.gpu
@pytest.mark.parametrize("n,v,h,gw_dtype", [(20000, 3000, 256, F32), (20000, 3000, 265, None), (700, 70000, 136, F32)])
def test_long_sums_of_unlike_tokens_repeat(lib, n, v, h, gw_dtype):
    """Several runs and tokens with scales of their own: the same bits whatever the workspace held, and from a graph."""
    x, w, label = problem(n, v, h, F16, 23, ignored=0.1)
    gloss = torch.exp2(-20.0 * torch.rand(n, device="cuda", generator=gen(1)))
    loss, lse = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    lib.linear_softmax_loss(loss, lse, x, w, label)
    gx, gw = torch.empty_like(x), torch.empty(v, h, dtype=gw_dtype or F16, device="cuda")
    ws = torch.empty(lib.linear_softmax_loss_workspace(n, v, h, gradient=True), dtype=torch.uint8, device="cuda")

    def run():
        lib.linear_softmax_loss_grad(gx, gw, x, w, label, lse, gloss, 0.01, workspace=ws,
                                     stream=torch.cuda.current_stream().cuda_stream)

    seen = []
    for fill in (0, 0xff):
        ws.fill_(fill)
        run()
        seen.append((gx.clone(), gw.clone()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    ws.fill_(0xff)
    gx.fill_(9)
    gw.fill_(9)
    graph.replay()
    torch.cuda.synchronize()
    seen.append((gx, gw))
    for other in seen[1:]:
        assert torch.equal(other[0], seen[0][0]) and torch.equal(other[1], seen[0][1])
    assert torch.isfinite(gx).all() and torch.isfinite(gw).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("size", [3e38, 1e34, 1e-30, 2e-38])
def test_loss_grad_of_huge_and_tiny_gloss(lib, dtype, size):
    """gloss near the ends of binary32's range, undone by the scale."""
    x, w, label = problem(50, 300, 40, dtype, 4, ignored=0.1)
    gloss = torch.full((50,), size, device="cuda") * (0.5 + 0.5 * torch.rand(50, device="cuda", generator=gen(3)))
    check_grad(lib, x, w, label, gloss=gloss, scale=float(np.float32(0.25 / size)), gw_dtype=F32)
