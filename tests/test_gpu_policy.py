"""Log probabilities, entropy, alternatives and their gradient against the formulas in 64 bits: every type, row widths on both sides of every way to split
a row, rows at every alignment, masks, rows that nothing is left of, infinities, lowest values, ties, other streams, capture.

Tolerances, from the arithmetic (u = 2^-24): d = (x - m) c is off by at most 3 u |d|, e^d by (4 + 3 |d|) u relative, a sum of n positive terms in
which no term takes part in more than n/32 + 64 additions by that many u relative.  So log S is off by E = (n/32 + 70 + 3 |d|) u, where the terms that
count have |d| <= 3 + log n + |log p| ..., and the results by E times their own size and 1."""
import numpy as np
import pytest

import policy_plain as plain

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
U = 2.0 ** -24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def code(pkg, t):
    return {"f32": pkg.F32, "bf16": pkg.BF16, "f16": pkg.F16}[t]


def cuda(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def place(x, t, stride, offset):
    """x as the device array that a caller might have: rows `stride` values apart, the first `offset` values into a buffer; NaN in what lies between."""
    n, v = x.shape
    buffer = torch.full((offset + max(1, n) * stride + 8,), float("nan"), dtype=TYPES[t], device="cuda")
    view = buffer[offset:offset + max(1, n) * stride].view(max(1, n), stride)[:n, :v]
    view.copy_(torch.from_numpy(np.asarray(x, np.float64)).cuda().to(TYPES[t]))
    return buffer, view


def forward(pkg, view, t, taken, legal=None, scale=1.0, top=0, stats=False, stream=0):
    n, v = view.shape
    dev = view.device
    lp, h = (torch.full((n + 3,), 77.0, device=dev) for _ in range(2))
    ta, tl = torch.full((n * top + 3,), 77, dtype=torch.int32, device=dev), torch.full((n * top + 3,), 77.0, device=dev)
    st = torch.full((n + 1, 4), 77.0, device=dev)
    p = pkg.PolicyRows(view.data_ptr(), code(pkg, t), n, v, row_stride=view.stride(0) if n else v, legal=legal.data_ptr() if legal is not None else None,
                       legal_stride=0 if legal is None or legal.dim() == 1 else legal.stride(0), taken=taken.data_ptr() if taken is not None else None, inv_temperature=scale)
    pkg.policy_logprobs(p, lp.data_ptr() if taken is not None else None, h.data_ptr(), st.data_ptr() if stats else None, top, ta.data_ptr() if top else None,
                        tl.data_ptr() if top else None, stream)
    return p, (lp, h, ta, tl, st), (view, taken, legal)


def check_forward(pkg, x, t, taken, legal=None, scale=1.0, top=0, stride=None, offset=0, mask_stride=None):
    n, v = x.shape
    scale = float(np.float32(scale))
    _buffer, view = place(x, t, stride or v, offset)
    x = view.double().cpu().numpy()                                          # as rounded to the type
    mask = None
    if legal is not None:
        mask = cuda(legal.astype(np.uint8)) if legal.ndim == 1 else torch.full((n, mask_stride or v), 1, dtype=torch.uint8, device="cuda")
        if legal.ndim == 2:
            mask[:, :v] = cuda(legal.astype(np.uint8))
    _p, (lp, h, ta, tl, _st), _keep = forward(pkg, view, t, None if taken is None else cuda(taken.astype(np.int32)), mask, scale, top)
    elp, eh, eta, etl, logp = plain.logprobs(x, taken, legal, scale, top)
    ta, tl = ta.cpu().numpy(), tl.double().cpu().numpy()
    lp, h = lp.double().cpu().numpy(), h.double().cpu().numpy()
    assert (lp[n:] == 77).all() and (h[n:] == 77).all() and (ta[n * top:] == 77).all() and (tl[n * top:] == 77).all()
    assert taken is not None or (lp == 77).all()
    ta, tl = ta[:n * top].reshape(n, top), tl[:n * top].reshape(n, top)
    assert not (lp[:n] > 0).any() and not (h[:n] < 0).any() and not (tl > 0).any()
    e = (v / 32 + 70 + 3 * (12 + np.log(v))) * U
    if taken is not None:
        close(lp[:n], elp, e + 4 * U * np.abs(elp))
    close(h[:n], eh, e * (2 + np.abs(eh)))
    bad = np.isnan(eh)
    assert np.array_equal(ta[~bad], eta[~bad]) and (ta[bad] == -1).all()
    close(tl, etl, e + 4 * U * np.abs(etl))


def close(got, want, tol):
    fine = np.isfinite(want)
    assert np.array_equal(got[~fine], want[~fine], equal_nan=True)
    off = np.abs(got[fine] - want[fine])
    tol = np.broadcast_to(tol, want.shape)[fine]
    assert (off <= tol).all(), "off by %g where %g is allowed" % (off[np.argmax(off - tol)], tol[np.argmax(off - tol)])


def check_gradient(pkg, x, t, taken, gl, gh, legal=None, scale=1.0, stride=None, offset=0, grad_stride=None, grad_offset=0, in_place=False):
    n, v = x.shape
    scale = float(np.float32(scale))
    buffer, view = place(x, t, stride or v, offset)
    x = view.double().cpu().numpy()
    mask = cuda(legal.astype(np.uint8)) if legal is not None else None
    p, (_lp, _h, _ta, _tl, st), _keep = forward(pkg, view, t, None if taken is None else cuda(taken.astype(np.int32)), mask, scale, 0, True)
    if in_place:
        out_buffer, out = buffer, view
    else:
        out_buffer, out = place(np.zeros((n, v)), t, grad_stride or v, grad_offset)
    dgl, dgh = (None if g is None else cuda(g.astype(np.float32)) for g in (gl, gh))
    pkg.policy_logprobs_backward(p, st.data_ptr(), None if dgl is None else dgl.data_ptr(), None if dgh is None else dgh.data_ptr(), out.data_ptr(), out.stride(0))
    torch.cuda.synchronize()
    assert (st[n:] == 77).all()
    got = out.double().cpu().numpy()
    out.fill_(float("nan"))
    assert torch.isnan(out_buffer).all()                                     # nothing was written between the rows
    gl64, gh64 = (None if g is None else g.astype(np.float32).astype(np.float64) for g in (gl, gh))
    want = plain.gradient(x, taken, gl64, gh64, legal, scale)
    _lp, h, _a, _t, logp = plain.logprobs(x, taken, legal, scale)
    pr = np.exp(logp)
    e = (v / 32 + 70 + 3 * (12 + np.log(v)) + 8) * U
    size_l = np.zeros(n) if gl64 is None or taken is None else np.abs(gl64)
    size_h = np.zeros(n) if gh64 is None else np.abs(gh64)
    with np.errstate(invalid="ignore"):
        tol = scale * (size_l[:, None] * np.where(pr > 0, pr, 0) + size_h[:, None] * pr * (np.where(pr > 0, np.abs(logp), 0) + h[:, None] + 1)) * 2 * e
    # a probability below 2^-126 is no normal float and counts as 0: what it is multiplied by is what that can be off by
    with np.errstate(invalid="ignore"):
        tiny = 2.0 ** -126 * scale * np.nan_to_num(size_l[:, None] + size_h[:, None] * (np.where(pr > 0, np.abs(logp), 0) + h[:, None] + 1))
    tol = np.nan_to_num(tol) + tiny + np.nan_to_num(np.abs(want)) * (4 * U + plain.HALF_STEP[t]) + plain.TINY[t]
    close(got, want, tol)


def some(rng, n, v, spread=3.0):
    x = rng.standard_normal((n, v)) * spread * rng.random((n, 1)) + 5 * rng.standard_normal((n, 1))
    taken = rng.integers(0, v, n)
    taken[n // 2:n // 2 + 1] = -1
    return x, taken


WIDTHS = [1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 255, 256, 257, 511, 513, 1000, 1023, 1025, 2047, 2049, 4096, 4099, 8191, 8193, 16385, 33000, 65537]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("v", WIDTHS)
def test_widths(pkg, t, v):
    rng = np.random.default_rng(v)
    for n in ((1, 3, 130) if v < 5000 else (1, 5)):
        x, taken = some(rng, n, v)
        check_forward(pkg, x, t, taken, top=min(32, v))
        check_forward(pkg, x, t, taken, scale=0.7, stride=v + 5, offset=3)
        gl, gh = rng.standard_normal(n), rng.standard_normal(n) * 0.1
        check_gradient(pkg, x, t, taken, gl, gh)
        check_gradient(pkg, x, t, taken, gl, None, scale=1.7, stride=v + 3, offset=1, grad_stride=v + 2, grad_offset=5)
        check_gradient(pkg, x, t, None, None, gh, in_place=True, stride=v + 1)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("offset", range(9))
def test_alignments(pkg, t, offset):
    rng = np.random.default_rng(offset)
    for v, stride in ((4, 4), (6, 9), (40, 41), (130, 133), (2500, 2501), (9000, 9003)):
        x, taken = some(rng, 9, v)
        legal = rng.random((9, v)) < 0.6
        check_forward(pkg, x, t, taken, legal, top=3, stride=stride, offset=offset, mask_stride=v + offset)
        check_gradient(pkg, x, t, taken, rng.standard_normal(9), rng.standard_normal(9), stride=stride, offset=offset, grad_stride=v + 8 - offset, grad_offset=offset // 2)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("v", [4, 13, 70, 300, 3001, 20001])
def test_masks(pkg, t, v):
    rng = np.random.default_rng(v)
    n = 20
    x, taken = some(rng, n, v)
    legal = rng.random((n, v)) < 0.5
    legal[3] = False                                                         # nothing is left
    legal[4] = False; legal[4, v - 1] = True                                 # one action is left
    legal[5] = True
    hidden = np.where(legal, x, rng.choice([np.nan, np.inf, -np.inf, 60000.0], (n, v)))      # whatever is masked does not exist
    gl, gh = rng.standard_normal(n), rng.standard_normal(n)
    for top in (0, 5):
        check_forward(pkg, hidden, t, taken, legal, top=top, scale=1.3)
    check_gradient(pkg, hidden, t, taken, gl, gh, legal)
    one = rng.random(v) < 0.5
    check_forward(pkg, x, t, taken, one, top=min(v, 7))                      # one mask for all rows
    check_gradient(pkg, x, t, taken, gl, gh, one)
    check_forward(pkg, x, t, taken, np.zeros(v, bool), top=2)
    check_gradient(pkg, x, t, taken, gl, gh, np.zeros(v, bool))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("v", [4, 9, 40, 200, 1500, 9001])
def test_values_at_the_edges(pkg, t, v):
    """Minus infinity and the type's lowest value in some or all places, NaN and plus infinity, huge differences, rows of one value."""
    lowest = float(torch.finfo(TYPES[t]).min)
    rng = np.random.default_rng(v)
    x = rng.standard_normal((16, v)) * 2
    x[0] = -np.inf
    x[1] = lowest
    x[2] = lowest; x[2, v // 2] = 1.0
    x[3] = -np.inf; x[3, v - 1] = -2.0
    x[4] = lowest; x[4, ::2] = -np.inf
    x[5, v // 3] = np.nan
    x[6, v // 3] = np.inf
    x[7] = -np.inf; x[7, 1] = np.nan
    x[8] = 0.25
    x[9] = -lowest; x[9, ::3] = lowest
    x[10, ::2] = -np.inf
    x[11] *= 1000
    x[12] = np.where(rng.random(v) < 0.5, 0.0, -0.0)                         # equal: the lowest action first
    x[13] = lowest / 2; x[13, 1:] = lowest
    x[14] = 40.0; x[14, v // 2:] = -40.0
    x[15] = np.where(np.arange(v) < max(2, v // 5), x[15], -1e12 if t != "f16" else -60000.0)      # a mask of the caller's own making
    taken = rng.integers(0, v, 16)
    taken[2] = v // 2; taken[3] = v - 1
    for scale in (1.0, 0.5, 3.0):
        check_forward(pkg, x, t, taken, top=min(v, 6), scale=scale)
        gl, gh = rng.standard_normal(16), rng.standard_normal(16) * 0.1
        gl[9] = gh[9] = 0.01                                                 # (finite in every type)
        check_gradient(pkg, x, t, taken, gl, gh, scale=scale)
    check_forward(pkg, x, t, taken, np.ones((16, v), bool), top=min(v, 6))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("v", [6, 50, 256, 1200, 5000, 30011])
@pytest.mark.parametrize("top", [1, 2, 5, 31, 32])
def test_alternatives(pkg, t, v, top):
    """Ties at every place, rows in rising and falling order, all the large values in one stretch."""
    rng = np.random.default_rng(v * 100 + top)
    x = np.stack([rng.integers(0, 4, v) * 1.0, np.zeros(v), np.arange(v) / v * 8, -np.arange(v) / v * 8, np.where((np.arange(v) > v // 2) & (np.arange(v) < v // 2 + 100), 5.0 + rng.random(v), rng.random(v)),
                  rng.standard_normal(v), np.where(np.arange(v) % 256 == 7, 9.0, rng.random(v)), np.where(rng.random(v) < 4 / v, 1.0, -np.inf)])
    legal = rng.random(x.shape) < 0.9
    taken = rng.integers(0, v, len(x))
    check_forward(pkg, x, t, taken, top=top)                                 # (top may be more than there are)
    check_forward(pkg, x, t, taken, legal, top=top, stride=v + 1)


@pytest.mark.parametrize("t", TYPES)
def test_many_rows_and_one_long_row(pkg, t):
    rng = np.random.default_rng(5)
    for n, v in ((70001, 4), (33333, 5), (20011, 19), (5003, 150), (1, 200003), (2, 131072), (3, 400001), (200, 150001)):
        x = torch.randn(n, v, device="cuda", generator=torch.Generator("cuda").manual_seed(n)).to(TYPES[t])
        taken = torch.from_numpy(rng.integers(0, v, n).astype(np.int32)).cuda()
        p, (lp, h, ta, tl, st), _keep = forward(pkg, x, t, taken, top=2, stats=True)
        logp = torch.log_softmax(x.double(), 1)
        e = (v / 32 + 70 + 3 * (12 + np.log(v))) * U
        want = logp.gather(1, taken.long()[:, None])[:, 0]
        assert ((lp[:n] - want).abs() <= e + 4 * U * want.abs()).all()
        eh = -(logp.exp() * logp).sum(1)
        assert ((h[:n] - eh).abs() <= e * (2 + eh)).all()
        assert torch.equal(ta[:2 * n].view(n, 2)[:, 0].long(), (x == x.amax(1, keepdim=True)).int().argmax(1))
        gl, gh = torch.randn(n, device="cuda"), torch.randn(n, device="cuda")
        g = torch.empty(n, v, dtype=TYPES[t], device="cuda")
        pkg.policy_logprobs_backward(p, st.data_ptr(), gl.data_ptr(), gh.data_ptr(), g.data_ptr())
        pr = logp.exp()
        one = torch.zeros_like(pr).scatter_(1, taken.long()[:, None], 1.0)
        eg = gl[:, None] * (one - pr) - gh[:, None] * pr * (logp + eh[:, None])
        tol = (gl.abs()[:, None] * pr + gh.abs()[:, None] * pr * (logp.abs() + eh[:, None] + 1)) * 2 * (e + 8 * U) + eg.abs() * (4 * U + plain.HALF_STEP[t]) + plain.TINY[t]
        assert ((g.double() - eg).abs() <= tol).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("n,v,top", [(1300, 1025, 3), (1300, 2500, 32), (1201, 5003, 8), (1184, 8192, 1), (310, 9001, 5), (700, 33000, 2), (80, 70001, 20), (2500, 300, 4), (9001, 700, 1),
                                     (4099, 1024, 16), (30000, 33, 6), (5, 131072, 32)])
def test_every_way_to_split_the_work(pkg, t, masked, n, v, top):
    """Many rows and few of them, a warp, a block or a cluster each: against 64 bits on the device, with rows that nothing is left of among the others."""
    gen = torch.Generator("cuda").manual_seed(n + v)
    x = (torch.randn(n, v, device="cuda", generator=gen) * 3).to(TYPES[t])
    legal = None
    z = x.double() * float(np.float32(0.8))
    if masked:
        legal = torch.rand(n, v, device="cuda", generator=gen) < 0.4
        legal[n // 2] = False
        legal[3] = False
        legal[3, v - 1] = True
        z = z.masked_fill(~legal, -np.inf)
        legal = legal.to(torch.uint8)
    taken = torch.randint(0, v, (n,), device="cuda", dtype=torch.int32, generator=gen)
    p, (lp, h, ta, tl, st), _keep = forward(pkg, x, t, taken, legal, 0.8, top, stats=True)
    empty = torch.isinf(z).all(1)
    logp = (z - torch.logsumexp(z, 1, keepdim=True)).masked_fill(empty[:, None], -np.inf)
    pr = logp.exp()
    e = (v / 32 + 70 + 3 * (12 + np.log(v))) * U
    want = logp.gather(1, taken.long()[:, None])[:, 0]
    assert torch.equal(torch.isinf(want), torch.isinf(lp[:n]))
    fine = ~torch.isinf(want)
    assert ((lp[:n] - want)[fine].abs() <= e + 4 * U * want[fine].abs()).all()
    eh = -torch.nan_to_num(pr * logp, nan=0.0).sum(1)
    assert ((h[:n] - eh).abs() <= e * (2 + eh)).all()
    key = x.double() if legal is None else x.double().masked_fill(legal == 0, -np.inf)
    best, at = torch.sort(key, dim=1, descending=True, stable=True)
    at = at[:, :top].masked_fill(torch.isinf(best[:, :top]), -1)
    assert torch.equal(ta[:n * top].view(n, top).long(), at)
    wl = logp.gather(1, at.clamp(min=0)).masked_fill(at < 0, -np.inf)
    tl = tl[:n * top].view(n, top)
    assert torch.equal(torch.isinf(tl), torch.isinf(wl))
    fine = ~torch.isinf(wl)
    assert ((tl - wl)[fine].abs() <= e + 4 * U * wl[fine].abs()).all()
    gl, gh = torch.randn(n, device="cuda", generator=gen), torch.randn(n, device="cuda", generator=gen)
    g = torch.empty(n, v, dtype=TYPES[t], device="cuda")
    pkg.policy_logprobs_backward(p, st.data_ptr(), gl.data_ptr(), gh.data_ptr(), g.data_ptr())
    one = torch.zeros_like(pr).scatter_(1, taken.long()[:, None], 1.0)
    lq = torch.where(pr > 0, logp, 0.0)
    scale = float(np.float32(0.8))
    eg = scale * (gl[:, None] * (one - pr) - gh[:, None] * pr * (lq + eh[:, None]))
    eg[empty] = 0.0
    if legal is not None:
        eg[legal == 0] = 0.0
    tol = scale * (gl.abs()[:, None] * pr + gh.abs()[:, None] * pr * (lq.abs() + eh[:, None] + 1)) * 2 * (e + 8 * U) + eg.abs() * (4 * U + plain.HALF_STEP[t]) + plain.TINY[t]
    assert ((g.double() - eg).abs() <= tol).all()


def test_rows_far_apart(pkg):
    """Offsets above 32 bits: three rows 2^31 values apart."""
    v, stride = 1003, (1 << 31) + 8
    buffer = torch.empty(2 * stride + v, dtype=torch.bfloat16, device="cuda")
    x = torch.randn(3, v, device="cuda").bfloat16()
    for r in range(3):
        buffer[r * stride:r * stride + v] = x[r]
    taken = torch.tensor([5, 1002, 0], dtype=torch.int32, device="cuda")
    p, (lp, h, ta, _tl, st), _keep = forward(pkg, torch.as_strided(buffer, (3, v), (stride, 1)), "bf16", taken, top=1, stats=True)
    want = torch.log_softmax(x.double(), 1).gather(1, taken.long()[:, None])[:, 0]
    assert ((lp[:3] - want).abs() <= (v / 32 + 130) * U + 4 * U * want.abs()).all()
    gl = torch.ones(3, device="cuda")
    pkg.policy_logprobs_backward(p, st.data_ptr(), gl.data_ptr(), None, buffer.data_ptr(), stride)      # in place
    pr = torch.softmax(x.double(), 1)
    for r in range(3):
        want = torch.nn.functional.one_hot(taken[r].long(), v) - pr[r]
        assert ((buffer[r * stride:r * stride + v].double() - want).abs() <= want.abs() * 2.0 ** -8 * 1.01 + 1e-9).all()


def test_no_rows_and_single_outputs(pkg):
    p = pkg.PolicyRows(0, pkg.F32, 0, 4)
    pkg.policy_logprobs(p)
    x, taken = torch.randn(50, 30, device="cuda"), torch.randint(0, 30, (50,), device="cuda", dtype=torch.int32)
    _p, every, _keep = forward(pkg, x, "f32", taken, top=4, stats=True)
    _p, some_, _keep = forward(pkg, x, "f32", None, top=4)
    assert all(torch.equal(a, b) for a, b in zip(every[1:4], some_[1:4])) and (some_[0] == 77).all()
    lp = torch.empty(50, device="cuda")
    pkg.policy_logprobs(pkg.PolicyRows(x.data_ptr(), pkg.F32, 50, 30, taken=taken.data_ptr()), lp.data_ptr())
    assert torch.equal(lp, every[0][:50])


def test_host_arrays_are_refused(pkg):
    x, taken = torch.randn(4, 4, device="cuda"), torch.zeros(4, dtype=torch.int32)
    out = torch.empty(4, device="cuda")
    with pytest.raises(pkg.CudarlError, match="taken is not device memory"):
        pkg.policy_logprobs(pkg.PolicyRows(x.data_ptr(), pkg.F32, 4, 4, taken=taken.data_ptr()), out.data_ptr())
    with pytest.raises(pkg.CudarlError, match="logits is not device memory"):
        pkg.policy_logprobs(pkg.PolicyRows(x.cpu().pin_memory().data_ptr(), pkg.F32, 4, 4), None, out.data_ptr())


@pytest.mark.parametrize("v", [4, 90, 5000, 150001])
def test_capture_and_other_streams(pkg, v):
    """Two graphs on two streams, replayed at once with new contents in the same places, and calls with none of them in between."""
    n = 7
    x = [torch.randn(n, v, device="cuda") for _ in range(2)]
    taken = torch.randint(0, v, (n,), device="cuda", dtype=torch.int32)
    gl, gh = torch.randn(n, device="cuda"), torch.randn(n, device="cuda")

    def both(k, stream, keep):
        p, out, more = forward(pkg, x[k], "f32", taken, top=3, stats=True, stream=stream)
        g = torch.empty_like(x[k])
        pkg.policy_logprobs_backward(p, out[4].data_ptr(), gl.data_ptr(), gh.data_ptr(), g.data_ptr(), stream=stream)
        keep.append((p, out, more, g))

    graphs, keeps = [], []
    for k in range(2):
        g, keep = torch.cuda.CUDAGraph(), []
        with torch.cuda.graph(g):
            both(k, torch.cuda.current_stream().cuda_stream, keep)
        graphs.append(g); keeps.append(keep)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for t in x:
            t.normal_()
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for k in range(2):
            keep = []
            both(k, 0, keep)
            torch.cuda.synchronize()
            assert torch.equal(keep[0][3], keeps[k][0][3])
            assert all(torch.equal(a, b) for a, b in zip(keep[0][1], keeps[k][0][1]))


def test_gradient_against_differences(pkg):
    """The loss sum(gl logprob + gh entropy) of the forward call itself, moved along single logits."""
    rng = np.random.default_rng(1)
    n, v = 4, 11
    x, taken = some(rng, n, v)
    x = x.astype(np.float32)
    gl, gh = rng.standard_normal(n), rng.standard_normal(n)

    def loss(y):
        _b, view = place(y, "f32", v, 0)
        _p, (lp, h, *_), _k = forward(pkg, view, "f32", cuda(taken.astype(np.int32)))
        return gl * lp[:n].double().cpu().numpy() + gh * h[:n].double().cpu().numpy()

    p, out, _keep = forward(pkg, place(x, "f32", v, 0)[1], "f32", cuda(taken.astype(np.int32)), stats=True)
    _b, view = place(x, "f32", v, 0)
    p.logits = view.data_ptr()
    g = torch.empty(n, v, device="cuda")
    dgl, dgh = cuda(gl.astype(np.float32)), cuda(gh.astype(np.float32))
    pkg.policy_logprobs_backward(p, out[4].data_ptr(), dgl.data_ptr(), dgh.data_ptr(), g.data_ptr())
    g = g.double().cpu().numpy()
    step = 2.0 ** -6
    for j in range(v):
        up, down = x.copy(), x.copy()
        up[:, j] += step; down[:, j] -= step
        d = (loss(up) - loss(down)) / (up[:, j].astype(np.float64) - down[:, j].astype(np.float64))
        # third derivatives of log p and H are at most 1 and 6 + 2 H (H <= log 11); outputs are off by 2^-16 at most
        assert (np.abs(d - g[:, j]) <= (np.abs(gl) + 11 * np.abs(gh)) * (step ** 2 / 6 + 2.0 ** -16 / step)).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("v", [1, 4, 33, 127, 128, 129])
def test_gradients_of_short_rows_without_statistics(pkg, t, v):
    """Up to 128 actions: neither written nor read, so that None, or any address, gives the same gradient; from 129 on they are needed."""
    n = 37
    x, taken = torch.randn(n, v, device="cuda").to(TYPES[t]), torch.randint(0, v, (n,), device="cuda", dtype=torch.int32)
    gl, gh = torch.randn(n, device="cuda"), torch.randn(n, device="cuda")
    p, out, _keep = forward(pkg, x, t, taken, stats=True)
    grads = [torch.full_like(x, 77) for _ in range(3)]
    pkg.policy_logprobs_backward(p, out[4].data_ptr(), gl.data_ptr(), gh.data_ptr(), grads[0].data_ptr())
    torch.cuda.synchronize()
    if v > pkg.ACTIONS_WITHOUT_STATS:
        with pytest.raises(pkg.CudarlError, match="stats"):
            pkg.policy_logprobs_backward(p, None, gl.data_ptr(), gh.data_ptr(), grads[1].data_ptr())
        with pytest.raises(pkg.CudarlError, match="stats is not aligned"):
            pkg.policy_logprobs_backward(p, out[4].data_ptr() + 4, gl.data_ptr(), gh.data_ptr(), grads[1].data_ptr())
        return
    assert (out[4] == 77).all()
    pkg.policy_logprobs_backward(p, None, gl.data_ptr(), gh.data_ptr(), grads[1].data_ptr())
    pkg.policy_logprobs_backward(p, 4, gl.data_ptr(), gh.data_ptr(), grads[2].data_ptr())
    assert torch.equal(grads[0], grads[1]) and torch.equal(grads[0], grads[2])


# rows and actions for every way to split the work: single lanes, teams, a warp, 128 threads, clusters of 2, 4 and 8 blocks (which of them goes by the type, too)
SPLITS = [(1500, 4), (1500, 100), (1500, 257), (3000, 700), (1300, 2500), (1200, 8191), (400, 5003), (400, 9001), (300, 33001), (140, 20001), (70, 40003), (7, 70001), (2, 131075)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("top", [0, 3])
@pytest.mark.parametrize("n,v", SPLITS)
def test_one_value_in_every_chunk(pkg, t, masked, top, n, v):
    """A row that holds one value -- all others are minus infinity, or masked -- which is in turn at either end and in every chunk of 16 bytes, in rows at every alignment:
    a value that is left out leaves nothing, one that counts twice halves the probability; in the gradient every place is written once."""
    rng = np.random.default_rng(v)
    per = 4 if t == "f32" else 8
    places = np.concatenate([np.arange(min(v, 40)), np.arange(max(0, v - 40), v), np.arange(0, v - per, per) + np.arange(len(range(0, v - per, per))) % per]) if v > 1100 else np.arange(v)
    places = np.concatenate([places, rng.integers(0, v, -len(places) % n)])
    stride = v + 1
    buffer = torch.full((3 + n * stride,), 0.5 if masked else -np.inf, dtype=TYPES[t], device="cuda")
    view = torch.as_strided(buffer, (n, v), (stride, 1), 3)
    legal = torch.zeros(n, v + 1, dtype=torch.uint8, device="cuda")[:, :v] if masked else None
    gl, one = torch.ones(n, device="cuda"), torch.ones(n, 1, device="cuda")
    grad = torch.empty(n, v, dtype=TYPES[t], device="cuda")
    fails = torch.zeros((), dtype=torch.int64, device="cuda")
    for at in range(0, len(places), n):
        j = torch.from_numpy(places[at:at + n].astype(np.int32)).cuda()
        jl = j.long()[:, None]
        if masked:
            legal.scatter_(1, jl, 1)
        else:
            view.scatter_(1, jl, 0.5)
        _p, (lp, h, ta, tl, _st), _keep = forward(pkg, view, t, j, legal, top=top)
        fails += (~(lp[:n].abs() <= 1e-6)).sum() + (~(h[:n].abs() <= 1e-6)).sum()
        if top:
            fails += (ta[:n * top].view(n, top)[:, 0] != j).sum() + (ta[:n * top].view(n, top)[:, 1:] != -1).sum() + (~(tl[:n * top].view(n, top)[:, 0].abs() <= 1e-6)).sum()
        else:
            other = (j + 1 + v // 3) % v                                     # the action taken is one without any probability: 1 there, -1 where the value is
            p, (_lp, _h, _ta, _tl, st), _keep = forward(pkg, view, t, other, legal, stats=True)
            grad.fill_(77)
            pkg.policy_logprobs_backward(p, st.data_ptr(), gl.data_ptr(), None, grad.data_ptr())
            g = grad.float()
            g.scatter_add_(1, jl, one)
            if not masked:
                g.scatter_add_(1, other.long()[:, None], -one)
            fails += (~(g.abs() <= 1e-6)).sum()
        if masked:
            legal.scatter_(1, jl, 0)
        else:
            view.scatter_(1, jl, -np.inf)
    assert int(fails) == 0


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("n,v", [s for s in SPLITS if s[1] > 1024])
def test_long_rows_within_the_error_of_their_longest_chain(pkg, t, masked, n, v):
    """Ordinary logits, with less room than a lost chunk of 16 bytes would take on the average.  A thread has at most v / (threads of a row) + 64 values, in two sums, and
    three roundings for every batch of 16 values or more; a dozen joins; a term is off by (4 + 3 |d|) u with |d| below 10 + log v for those that count."""
    per, blocks = (4 if t == "f32" else 8), 1
    while blocks < 8 and n * blocks < 2 * 148 and v >= 256 * per * 4 * blocks:
        blocks *= 2
    threads = 256 * blocks if blocks > 1 else 32 if v <= 8192 and n >= 8 * 148 else 128
    gen = torch.Generator("cuda").manual_seed(n + v)
    x = torch.randn(n, v, device="cuda", generator=gen).to(TYPES[t])
    z = x.double()
    legal = None
    if masked:
        legal = torch.rand(n, v, device="cuda", generator=gen) < 0.7
        z = z.masked_fill(~legal, -np.inf)
        legal = legal.to(torch.uint8)
    taken = torch.randint(0, v, (n,), device="cuda", dtype=torch.int32, generator=gen)
    p, (lp, h, _ta, _tl, st), _keep = forward(pkg, x, t, taken, legal, stats=True)
    logp = torch.log_softmax(z, 1)
    pr = logp.exp()
    chain = v / threads + 64
    e = (chain / 2 + 3 * chain / 16 + 12 + 4 + 3 * (10 + np.log(v))) * U
    assert e < per / v / 2
    want = logp.gather(1, taken.long()[:, None])[:, 0]
    fine = ~torch.isinf(want)
    assert torch.equal(~fine, torch.isinf(lp[:n])) and ((lp[:n] - want)[fine].abs() <= e + 4 * U * want[fine].abs()).all()
    lq = torch.where(pr > 0, logp, 0.0)
    eh = -(pr * lq).sum(1)
    assert ((h[:n] - eh).abs() <= e * (2 + eh)).all()
    gl, gh = torch.randn(n, device="cuda", generator=gen), torch.randn(n, device="cuda", generator=gen) * 0.1
    g = torch.empty(n, v, dtype=TYPES[t], device="cuda")
    pkg.policy_logprobs_backward(p, st.data_ptr(), gl.data_ptr(), gh.data_ptr(), g.data_ptr())
    eg = gl[:, None] * (torch.zeros_like(pr).scatter_(1, taken.long()[:, None], 1.0) - pr) - gh[:, None] * pr * (lq + eh[:, None])
    if masked:
        eg[legal == 0] = 0.0
    tol = pr * (gl.abs()[:, None] + gh.abs()[:, None] * (lq.abs() + eh[:, None] + 1)) * 2 * (e + 8 * U) + eg.abs() * (4 * U + plain.HALF_STEP[t]) + plain.TINY[t]
    assert ((g.double() - eg).abs() <= tol).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("v", [4, 9, 40, 200, 1500, 9001, 70001])
@pytest.mark.parametrize("scale", [1e-6, 1e-3, 1e3, 1e6])
def test_temperatures_at_their_ends(pkg, t, v, scale):
    """Rows on both sides of where differences are taken exactly, masks of the lowest value among them."""
    rng = np.random.default_rng(v)
    x, taken = some(rng, 12, v)
    if t != "f16":
        x[3] *= 1e4
        x[4] = rng.standard_normal(v) * 1e7
    x[5] = rng.standard_normal(v) * 1e-4
    x[6] = float(torch.finfo(TYPES[t]).min); x[6, v // 2] = 1.0
    x[7] = -np.inf; x[7, 0] = 2.5
    legal = rng.random((12, v)) < 0.6
    gl, gh = rng.standard_normal(12) / max(scale, 1), rng.standard_normal(12) * 0.1 / max(scale, 1)
    for mask in (None, legal):
        check_forward(pkg, x, t, taken, mask, scale=scale, top=min(v, 5))
        check_gradient(pkg, x, t, taken, gl, gh, mask, scale=scale)


@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_the_longest_row(pkg, t):
    """2^30 actions: one that has all the probability, at the ends and in the middle, and all of them alike (sums of ones are exact up to 2^24 a thread)."""
    v = 1 << 30
    x = torch.full((1, v), -np.inf, dtype=TYPES[t], device="cuda")
    grad = torch.empty(1, v, dtype=TYPES[t], device="cuda")
    gl = torch.ones(1, device="cuda")
    for j in (0, 1, (1 << 29) - 1, 1 << 29, v - 5, v - 1):
        x[0, j] = 1.5
        taken = torch.tensor([j], dtype=torch.int32, device="cuda")
        _p, (lp, h, ta, tl, _st), _keep = forward(pkg, x, t, taken, top=1)
        assert float(lp[0]) == 0.0 and float(h[0]) == 0.0 and int(ta[0]) == j and float(tl[0]) == 0.0
        other = (j + v // 2) % v
        p, (lp, _h, _ta, _tl, st), _keep = forward(pkg, x, t, torch.tensor([other], dtype=torch.int32, device="cuda"), stats=True)
        pkg.policy_logprobs_backward(p, st.data_ptr(), gl.data_ptr(), None, grad.data_ptr())
        assert float(lp[0]) == -np.inf and float(grad[0, j]) == -1.0 and float(grad[0, other]) == 1.0
        grad[0, j] = grad[0, other] = 0.0
        assert not bool(grad.any())
        x[0, j] = -np.inf
    x.fill_(0.25)
    _p, (lp, h, _ta, _tl, _st), _keep = forward(pkg, x, t, torch.tensor([v - 1], dtype=torch.int32, device="cuda"))
    want = 30 * np.log(2.0)
    assert abs(float(lp[0]) + want) <= 4 * U * want and abs(float(h[0]) - want) <= 4 * U * want
