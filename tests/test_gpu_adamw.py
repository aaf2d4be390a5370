"""AdamW over many tensors against the formula in 64 bits: every mixture of types, odd sizes and alignments, moments of 32 and 8 bits (the codes themselves,
rounded as the random stream says), clipping, steps that do not happen, capture, resumed runs -- and a policy trained on the arena with it.

Tolerances (u = 2^-24): m' has three roundings, v' four, the step a dozen on top of theirs; the new weight is rounded once more, and to its type."""
import ctypes as C

import numpy as np
import pytest

import policy_plain as plain

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
U = 2.0 ** -24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
TAG = 0x4F50544D


def code(pkg, t):
    return {"f32": pkg.F32, "bf16": pkg.BF16, "f16": pkg.F16}[t]


class Net:
    """Tensors of the sizes given, each in a buffer of its own `offset` values in, with sentinels around."""

    def __init__(self, pkg, sizes, param="f32", grad="f32", master=False, bits=32, offset=0, decay=0.01, seed=0, size=1e-2):
        gen = torch.Generator("cuda").manual_seed(seed)
        self.pkg, self.sizes, self.bits, self.offset, self.decay, self.all = pkg, sizes, bits, offset, decay, []
        self.master = master
        self.tensors = []
        for i, n in enumerate(sizes):
            def buffer(dtype, values):
                off = offset
                whole = torch.full((n + off + 40,), 77, device="cuda").to(dtype) if dtype != torch.uint8 else torch.full((n + off + 40,), 77, dtype=torch.uint8, device="cuda")
                whole[off:off + n] = values.to(dtype)
                self.all.append((whole, off, n))
                return whole[off:off + n]
            w = torch.randn(n, device="cuda", generator=gen)
            t = dict(param=buffer(TYPES[param], w), grad=buffer(TYPES[grad], torch.randn(n, device="cuda", generator=gen) * size * (i + 1)))
            if master:
                t["master"] = buffer(torch.float32, w)
            if bits == 32:
                t["m"] = buffer(torch.float32, torch.randn(n, device="cuda", generator=gen) * size)
                t["v"] = buffer(torch.float32, torch.rand(n, device="cuda", generator=gen) * size * size)
            else:
                blocks = (n + 255) // 256
                t["m"] = buffer(torch.uint8, torch.randint(0, 256, (n,), device="cuda", generator=gen))
                t["m"][(t["m"] & 127) == 127] = 126                          # no NaN
                t["v"] = buffer(torch.uint8, torch.randint(0, 127, (n,), device="cuda", generator=gen))
                for key in ("s1", "s2"):
                    whole = torch.full((blocks + 8,), 77.0, device="cuda")
                    whole[:blocks] = (0.5 + torch.rand(blocks, device="cuda", generator=gen)) * size / 448
                    self.all.append((whole, 0, blocks))
                    t[key] = whole[:blocks]
            self.tensors.append(t)
        self.param, self.grad = param, grad

    def list(self):
        p = lambda t, k: t[k].data_ptr() if k in t and t[k].numel() else None      # noqa: E731
        return [self.pkg.AdamWTensor(count=n, param=p(t, "param"), param_type=code(self.pkg, self.param), grad=p(t, "grad"), grad_type=code(self.pkg, self.grad), master=p(t, "master"),
                                     moment1=p(t, "m"), moment2=p(t, "v"), scale1=p(t, "s1"), scale2=p(t, "s2"), lr_scale=1.0 + 0.5 * (i % 2), weight_decay=self.decay * (i % 3))
                for i, (t, n) in enumerate(zip(self.tensors, self.sizes))]

    def moments(self, t):
        if self.bits == 32:
            return t["m"].double().cpu().numpy(), t["v"].double().cpu().numpy()
        value = np.concatenate([plain.E4M3, [np.nan], -plain.E4M3, [np.nan]])
        n = len(t["m"])
        s1, s2 = (t[k].double().cpu().numpy().repeat(256)[:n] for k in ("s1", "s2"))
        return value[t["m"].cpu().numpy()] * s1, (value[t["v"].cpu().numpy()] * s2) ** 2

    def snapshot(self):
        return [(t["master" if self.master else "param"].double().cpu().numpy(), t["grad"].double().cpu().numpy(), *self.moments(t)) for t in self.tensors]

    def untouched(self):
        for whole, off, n in self.all:
            edge = torch.cat([whole[:off], whole[off + n:]]).float()
            assert (edge == 77).all()


def check(net, before, step, lr, clip=1.0, seed=0, beta1=0.9, beta2=0.999):
    """What the tensors hold now against one step from `before` in 64 bits; returns how many codes there were that a rounding error of the value could decide."""
    first, unsure, n_all = 0, 0, 0
    for i, (t, (w, g, m, v)) in enumerate(zip(net.tensors, before)):
        n = len(w)
        lr_scale, decay = float(np.float32(1.0 + 0.5 * (i % 2))), float(np.float32(net.decay * (i % 3)))
        ew, em, ev = plain.adamw(w, g, m, v, step, float(np.float32(lr)), decay, clip, beta1, beta2, lr_scale=lr_scale)
        tol_m = 4 * U * (beta1 * np.abs(m) + (1 - beta1) * np.abs(g * clip)) + 1e-37
        tol_step = np.abs(ew - w) * 20 * U + lr * lr_scale * 4 * tol_m / np.maximum(np.sqrt(ev), 1e-30) / (1 - beta1 ** step) * np.sqrt(1 - beta2 ** step) + 2 * U * np.abs(ew) + U * lr * decay * np.abs(w)
        weight = t["master" if net.master else "param"].double().cpu().numpy()
        kept = "f32" if net.master else net.param
        assert (np.abs(weight - ew) <= tol_step + (0 if kept == "f32" else plain.HALF_STEP[kept] * np.abs(ew) + plain.TINY[kept])).all()
        if net.master:                                                       # the copy: the master, rounded
            assert torch.equal(t["param"], t["master"].to(TYPES[net.param]))
        if net.bits == 32:
            assert (np.abs(t["m"].double().cpu().numpy() - em) <= tol_m).all()
            assert (np.abs(t["v"].double().cpu().numpy() - ev) <= 5 * U * ev + 1e-37).all()
        else:
            blocks = (n + 255) // 256
            pad = blocks * 256 - n
            words = plain.philox(np.arange(first * 64, (first + blocks) * 64), step, seed, TAG).reshape(-1)[:n]
            for key, scale, x, bits in (("m", "s1", em, words & np.uint64(0xFFFF)), ("v", "s2", np.sqrt(ev), words >> np.uint64(16))):
                high = np.abs(np.concatenate([x, np.zeros(pad)])).reshape(-1, 256).max(1) / 448
                got = t[scale].double().cpu().numpy()
                assert (np.abs(got - high) <= 16 * U * high + 1e-38).all()
                y = np.minimum(np.abs(x) / np.where(got > 0, got, 1.0).repeat(256)[:n], 448.0)
                low = np.searchsorted(plain.E4M3, y, side="right") - 1
                step_ = np.where(low < 126, plain.E4M3[np.minimum(low + 1, 126)] - plain.E4M3[low], 32.0)
                part = (y - plain.E4M3[low]) / step_ + bits.astype(np.float64) / 65536 - 1   # >= 0: up
                want = np.minimum(low + (part >= 0), 126)
                if key == "v":
                    want = np.where((want == 0) & (x > 0), 1, want)
                codes = t[key].cpu().numpy()
                sure = np.abs(part) > 2.0 ** -16 + 64 * U * np.maximum(1, y / step_)      # 16 random bits against the kept 23: one part in 2^16 is either
                sure &= np.abs(part + 1) > 64 * U * np.maximum(1, y / step_)
                assert np.array_equal((codes & 127)[sure], want[sure])
                assert (np.abs((codes & 127).astype(int) - want) <= 1).all()
                assert np.array_equal(codes[want > 0] >= 128, x[want > 0] < 0)
                unsure += (~sure).sum(); n_all += n
            first += blocks
    assert unsure <= 0.002 * n_all + 4
    net.untouched()


SIZES = [1, 255, 256, 257, 7, 5000, 1024, 0, 33333, 2048, 13]


@pytest.mark.parametrize("param,master", [("f32", False), ("f32", True), ("bf16", False), ("bf16", True), ("f16", False), ("f16", True)])
@pytest.mark.parametrize("grad", TYPES)
@pytest.mark.parametrize("bits", [32, 8])
def test_types(pkg, param, master, grad, bits):
    net = Net(pkg, SIZES, param, grad, master, bits)
    opt = pkg.AdamW(net.list(), state_bits=bits, seed=(5 << 32) + 9, step=10)
    for step in (11, 12):
        before = net.snapshot()
        opt.step(0.01)
        check(net, before, step, 0.01, seed=(5 << 32) + 9)
    assert opt.get_stats().step == 12


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("offset", [1, 2, 3, 4, 5, 8, 12, 16])
def test_alignments(pkg, bits, offset):
    net = Net(pkg, [4097, 300, 8, 1500], "bf16", "f16", True, bits, offset=offset)
    before = net.snapshot()
    pkg.AdamW(net.list(), state_bits=bits).step(0.003)
    check(net, before, 1, 0.003)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("grad", TYPES)
@pytest.mark.parametrize("offset", [1, 2, 4, 8, 12])
@pytest.mark.parametrize("sizes", [[4097, 300, 8, 1500], [1500000, 2048, 7]])
def test_the_norm_of_gradients_at_every_alignment(pkg, bits, grad, offset, sizes):
    """Four values are 16 bytes in, where a bulk copy of them can start and eight of 32 bits cannot be loaded at once; few pieces, and more than blocks."""
    net = Net(pkg, sizes, "f32", grad, False, bits, size=1e-3)
    for t, n in zip(net.tensors, sizes):                                     # only the gradient lies oddly
        whole = torch.full((n + offset + 40,), 77, device="cuda").to(TYPES[grad])
        whole[offset:offset + n] = t["grad"]
        t["grad"] = whole[offset:offset + n]
        net.all.append((whole, offset, n))
    before = net.snapshot()
    norm = np.sqrt(sum((g ** 2).sum() for _w, g, _m, _v in before))
    most = float(np.float32(norm / 3))
    opt = pkg.AdamW(net.list(), state_bits=bits, max_grad_norm=most)
    opt.step(0.01)
    check(net, before, 1, 0.01, most / (norm + 1e-6))
    assert abs(opt.get_stats().grad_norm - norm) <= 1e-12 * norm
    net.untouched()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("grad", TYPES)
def test_clipping(pkg, bits, grad):
    net = Net(pkg, [100, 20000, 1, 777], grad=grad, bits=bits)
    for most, scale in ((1.0, 1.0), (1e6, 0.5), (0.25, -2.0)):
        before = net.snapshot()
        norm = np.sqrt(sum((g ** 2).sum() for _w, g, _m, _v in before)) * abs(scale)
        opt = pkg.AdamW(net.list(), state_bits=bits, max_grad_norm=most, seed=3)
        opt.step(0.01, grad_scale=scale)
        clip = min(1.0, most / (norm + 1e-6)) * scale
        check(net, before, 1, 0.01, clip, seed=3)
        s = opt.get_stats()
        assert abs(s.grad_norm - norm) <= 1e-12 * norm and (s.step, s.skipped) == (1, 0)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("bad", [np.inf, np.nan])
def test_a_step_that_does_not_happen(pkg, bits, bad):
    net = Net(pkg, [300, 5000], bits=bits)
    opt = pkg.AdamW(net.list(), state_bits=bits, max_grad_norm=1.0)
    opt.step(0.01)
    good = float(net.tensors[1]["grad"][4321])
    net.tensors[1]["grad"][4321] = bad
    whole = [a.clone() for a, _o, _n in net.all]
    opt.step(0.01)
    s = opt.get_stats()
    assert (s.step, s.skipped) == (1, 1) and not np.isfinite(s.grad_norm)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, (b, _o, _n) in zip(whole, net.all))
    net.tensors[1]["grad"][4321] = good
    before = net.snapshot()
    opt.step(0.01)
    norm = np.sqrt(sum((g ** 2).sum() for _w, g, _m, _v in before))
    check(net, before, 2, 0.01, min(1.0, 1.0 / (norm + 1e-6)))


def test_from_nothing_and_zero_gradients(pkg):
    """Moments of zeros (codes and scales too), tensors whose gradient is zero."""
    for bits in (32, 8):
        net = Net(pkg, [1000, 513], bits=bits)
        for t in net.tensors:
            for key in ("m", "v", "s1", "s2"):
                if key in t:
                    t[key].zero_()
        net.tensors[1]["grad"].zero_()
        opt = pkg.AdamW(net.list(), state_bits=bits, seed=8)
        for step in (1, 2, 3):
            before = net.snapshot()
            opt.step(0.01)
            check(net, before, step, 0.01, seed=8)
        assert not net.tensors[1]["m"].any() and not net.tensors[1]["v"].any()


def test_large_and_small_gradients_in_one_block(pkg):
    """A block over many orders of magnitude: a root that is not zero is never stored as zero, so no later step divides by eps alone."""
    net = Net(pkg, [512], bits=8)
    t = net.tensors[0]
    for key in ("m", "v", "s1", "s2"):
        t[key].zero_()
    t["grad"].copy_(torch.logspace(-12, 2, 512))
    opt = pkg.AdamW(net.list(), state_bits=8, seed=1)
    before = net.snapshot()
    opt.step(0.01)
    check(net, before, 1, 0.01, seed=1)
    assert (t["v"] > 0).all()
    w = t["param"].clone()
    t["grad"].zero_()
    opt.step(0.01)
    assert ((t["param"] - w).abs() <= 0.02).all()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("grad", ["f32", "bf16"])
@pytest.mark.parametrize("eps", [1e-30, 1e-8])
@pytest.mark.parametrize("n", [256, 255])
def test_gradients_over_a_floats_range(pkg, bits, grad, eps, n):
    """A tensor of `n` values (loaded wide, and one by one) for every decade from 1e-20, where v is a few steps of the subnormal floats, to 1e38, where it is infinite
    from 5.8e20 on; without clipping.  v is rounded by 2^-150 at the least, which is that much of its size and half as much of its root's; a root below 2^-50 is off by
    2^-22 more."""
    decades = list(range(-20, 39))
    net = Net(pkg, [n] * len(decades), grad=grad, bits=bits, decay=0.01)
    gen = torch.Generator("cuda").manual_seed(7)
    for t, d in zip(net.tensors, decades):
        for key in ("m", "v", "s1", "s2"):
            if key in t:
                t[key].zero_()
        g = (0.7 + 0.3 * torch.rand(n, device="cuda", generator=gen, dtype=torch.float64)) * 10.0 ** d
        t["grad"].copy_(g * (1 - 2 * torch.randint(0, 2, (n,), device="cuda", generator=gen)))
    before = net.snapshot()
    opt = pkg.AdamW(net.list(), state_bits=bits, eps=eps, seed=3)
    opt.step(0.01)
    eps, lr = float(np.float32(eps)), float(np.float32(0.01))
    for i, (t, (w, g, m, v), d) in enumerate(zip(net.tensors, before, decades)):
        lr_scale, decay = float(np.float32(1.0 + 0.5 * (i % 2))), float(np.float32(net.decay * (i % 3)))
        em, ev = 0.1 * g, 0.001 * g * g
        root = np.where(ev > plain.FLT_MAX, np.inf, np.sqrt(ev))
        off = 0.5 * (5 * U + 2.0 ** -150 / ev) + 2.0 ** -22                  # of the root
        step = lr * lr_scale * em / (1 - 0.9) / (root / np.sqrt(1 - 0.999) + eps)
        ew = w - lr * lr_scale * decay * w - step
        weight = t["param"].double().cpu().numpy()
        assert np.isfinite(weight).all(), d
        assert (np.abs(weight - ew) <= np.abs(step) * (24 * U + off) + 4 * U * np.abs(ew) + 4 * U * lr * decay * np.abs(w)).all(), d
        if bits == 32:
            got = t["v"].double().cpu().numpy()
            if d > 20:
                assert (got == np.inf).all()
            else:
                assert (np.abs(got - ev) <= 5 * U * ev + 2.0 ** -150).all()
            assert (np.abs(t["m"].double().cpu().numpy() - em) <= 4 * U * np.abs(em)).all()
        else:
            _m, got = net.moments(t)
            got = np.sqrt(got)
            kept = np.where(np.isinf(root), 2.0 ** 65, root)
            high = kept.max() / 448
            assert abs(float(t["s2"][0]) - high) <= (2 * U + off.max()) * high
            assert (np.abs(got - kept) <= kept * (2.0 ** -3 + off + 8 * U)).all()      # values within a factor of two of the block's largest: codes have three bits behind the first
    for t in net.tensors:
        t["grad"].zero_()
    still = [t["param"].clone() for t in net.tensors]
    opt.step(0.01)
    for i, (t, w, d) in enumerate(zip(net.tensors, still, decades)):
        assert torch.isfinite(t["param"]).all()
        if d > 20:                                                           # stays where it is
            w = w.double()
            assert ((t["param"].double() - w * (1 - lr * (1.0 + 0.5 * (i % 2)) * net.decay * (i % 3))).abs() <= 2 * U * w.abs()).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_one_gradient_beyond_the_range(pkg, bits):
    """Among ordinary ones: the others of its block take their step, nothing becomes NaN, zeros stay zeros."""
    net = Net(pkg, [700], bits=bits)
    t = net.tensors[0]
    for key in ("m", "v", "s1", "s2"):
        if key in t:
            t[key].zero_()
    t["grad"][5] = 3e30
    t["grad"][6] = 0.0
    before = net.snapshot()
    opt = pkg.AdamW(net.list(), state_bits=bits)
    opt.step(0.01)
    (w, g, m, v), = before
    ew, _m, _v = plain.adamw(w, g, m, v, 1, float(np.float32(0.01)), 0.0)
    ew[5] = w[5]
    got = t["param"].double().cpu().numpy()
    assert (np.abs(got - ew) <= 40 * U * 0.01 + 2 * U * np.abs(ew)).all()
    for _ in range(3):
        opt.step(0.01)
        assert torch.isfinite(t["param"]).all() and float(t["param"][5]) == float(w[5]) == got[5] and float(t["param"][6]) == float(w[6])
        assert bits == 8 or torch.isfinite(t["m"]).all()
        assert bits == 32 or (torch.isfinite(t["s1"]).all() and torch.isfinite(t["s2"]).all())


def test_many_tensors_and_a_large_one(pkg):
    sizes = [int(n) for n in np.random.default_rng(3).integers(1, 3000, 900)] + [3_000_001]
    for bits in (32, 8):
        net = Net(pkg, sizes, "bf16", "bf16", True, bits)
        before = net.snapshot()
        norm = np.sqrt(sum((g ** 2).sum() for _w, g, _m, _v in before))
        pkg.AdamW(net.list(), state_bits=bits, seed=2, max_grad_norm=0.5).step(0.01)
        check(net, before, 1, 0.01, 0.5 / (norm + 1e-6), seed=2)


@pytest.mark.parametrize("bits", [32, 8])
def test_two_handles_at_once(pkg, bits):
    """Two networks on two streams, and the same steps one after the other."""
    nets = [Net(pkg, [70000, 300, 5001], "bf16", "bf16", True, bits, seed=k % 2) for k in range(4)]
    opts = [pkg.AdamW(n.list(), state_bits=bits, seed=6, max_grad_norm=1.0) for n in nets]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for k in range(2):
            opts[k].step(0.01, stream=streams[k].cuda_stream)
    torch.cuda.synchronize()
    for k in (2, 3):
        for _ in range(20):
            opts[k].step(0.01)
    torch.cuda.synchronize()
    for k in range(2):
        for (a, _o, _n), (b, _o2, _n2) in zip(nets[k].all, nets[k + 2].all):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_no_tensors(pkg):
    opt = pkg.AdamW([])
    opt.step(0.1)
    assert opt.get_stats().step == 1
    opt = pkg.AdamW([], max_grad_norm=1.0)
    opt.step(0.1)
    assert (opt.get_stats().step, opt.get_stats().grad_norm) == (1, 0.0)


@pytest.mark.parametrize("bits", [32, 8])
def test_capture_counts_on(pkg, bits):
    """A captured step, replayed, is the same as as many calls."""
    nets = [Net(pkg, [3000, 50], "bf16", "bf16", True, bits) for _ in range(2)]
    opts = [pkg.AdamW(n.list(), state_bits=bits, seed=4, max_grad_norm=1.0) for n in nets]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        opts[0].step(0.01, stream=torch.cuda.current_stream().cuda_stream)
    for _ in range(7):
        g.replay()
        opts[1].step(0.01)
    torch.cuda.synchronize()
    assert opts[0].get_stats().step == opts[1].get_stats().step == 7
    for (a, _o, _n), (b, _o2, _n2) in zip(nets[0].all, nets[1].all):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("bits", [32, 8])
def test_a_resumed_run_goes_on_the_same(pkg, bits):
    nets = [Net(pkg, [3000, 50], bits=bits) for _ in range(2)]
    whole = pkg.AdamW(nets[0].list(), state_bits=bits, seed=4)
    for _ in range(6):
        whole.step(0.01)
    part = pkg.AdamW(nets[1].list(), state_bits=bits, seed=4)
    for _ in range(3):
        part.step(0.01)
    part = pkg.AdamW(nets[1].list(), state_bits=bits, seed=4, step=part.get_stats().step)
    for _ in range(3):
        part.step(0.01)
    torch.cuda.synchronize()
    # the powers of the betas: multiplied up or taken at once, the same to some 2^-52, which a float does not show but at a border
    same = [torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for (a, _o, _n), (b, _o2, _n2) in zip(nets[0].all, nets[1].all)]
    assert all(same)


def test_gradients_in_new_places(pkg):
    net = Net(pkg, [3000, 0, 50])
    opt = pkg.AdamW(net.list())
    grads = [torch.randn(n, device="cuda") * 0.01 for n in net.sizes]
    opt.set_gradients([g.data_ptr() for g in grads])
    for t, g in zip(net.tensors, grads):
        t["grad"].zero_()
    before = net.snapshot()
    before = [(w, g.double().cpu().numpy(), m, v) for (w, _g, m, v), g in zip(before, grads)]
    opt.step(0.01)
    check(net, before, 1, 0.01)
    with pytest.raises(pkg.CudarlError, match="null gradient"):
        opt.set_gradients([grads[0].data_ptr(), None, None])
    with pytest.raises(pkg.CudarlError, match="not device memory"):
        opt.set_gradients([torch.zeros(3000).data_ptr(), None, grads[2].data_ptr()])


def test_tensors_are_refused(pkg):
    net = Net(pkg, [100])
    def refused(word, bits=32, **kw):
        t = net.list()[0]
        for k, v in kw.items():
            setattr(t, k, v)
        with pytest.raises(pkg.CudarlError, match=word):
            pkg.AdamW([t], state_bits=bits)
    refused("count", count=-1)
    refused("null", param=None)
    refused("null", moment2=None)
    refused("scales", bits=8)
    refused("param_type", param_type=3)
    refused("grad_type", grad_type=-1)
    refused("weight_decay", weight_decay=float("nan"))
    refused("lr_scale", lr_scale=-1.0)
    refused("aligned", param=net.tensors[0]["param"].data_ptr() + 2)
    refused("not device memory", master=torch.zeros(100).data_ptr())
    refused("2\\^34", count=(1 << 34) + 1)                                   # (nothing of it is touched)
    t = net.list()[0]
    t.grad = None
    opt = pkg.AdamW([t])
    with pytest.raises(pkg.CudarlError, match="no gradient"):
        opt.step(0.1)
    opt.set_gradients([net.tensors[0]["grad"].data_ptr()])
    opt.step(0.1)
    for bad in (-1.0, float("nan"), float("inf")):
        with pytest.raises(pkg.CudarlError, match="lr"):
            opt.step(bad)
    with pytest.raises(pkg.CudarlError, match="grad_scale"):
        opt.step(0.1, grad_scale=float("nan"))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        s = torch.cuda.current_stream().cuda_stream
        with pytest.raises(pkg.CudarlError, match="captured"):
            opt.set_gradients([net.tensors[0]["grad"].data_ptr()], stream=s)
        opt.step(0.1, stream=s)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_policy_steps_the_arena_and_learns(pkg, bits):
    """All of it together: a policy (a table of logits over the cells, with a shared bias) chooses the moves of the arena's environments, the calls give log
    probabilities and entropies, the gradient of a policy-gradient loss, and the step of the weights; each quantity against 64 bits at every step."""
    w, h, n = 12, 9, 500
    world = pkg.VecGridWorld(pkg.make_config(w, h, n, 99, obstacle_kind=pkg.OBST_BERNOULLI, obstacle_p=0.1, goal_mode=pkg.GOAL_SEEDED, num_goals=1, start_mode=pkg.START_RANDOM))
    gen = torch.Generator("cuda").manual_seed(1)
    table, bias = torch.randn(w * h, 4, device="cuda", generator=gen) * 0.1, torch.zeros(4, device="cuda")
    tensors, keep, moments = [], [], []
    for p in (table, bias):
        g = torch.zeros_like(p)
        m, v = (torch.zeros(p.numel(), dtype=torch.uint8 if bits == 8 else torch.float32, device="cuda") for _ in range(2))
        s1, s2 = (torch.zeros((p.numel() + 255) // 256, device="cuda") for _ in range(2))
        keep.append(g); moments.append((m, v, s1, s2))
        tensors.append(pkg.AdamWTensor(count=p.numel(), param=p.data_ptr(), grad=g.data_ptr(), moment1=m.data_ptr(), moment2=v.data_ptr(), scale1=s1.data_ptr(), scale2=s2.data_ptr(),
                                       lr_scale=1.0, weight_decay=0.0))
    opt = pkg.AdamW(tensors, state_bits=bits, max_grad_norm=1.0)
    lib = pkg.load()
    rewards, dones = torch.zeros(n, device="cuda"), torch.zeros(n, dtype=torch.uint8, device="cuda")
    for step in range(8):
        x, y, _t = world.get_state()
        cell = torch.from_numpy(y.astype(np.int64) * w + x).cuda()
        logits = (table[cell] + bias).contiguous()
        noise = -torch.log(-torch.log(torch.rand(n, 4, device="cuda", generator=gen).clamp(1e-6, 1 - 1e-6)))
        taken = (logits + noise).argmax(1).int()
        torch.cuda.synchronize()
        assert lib.cudarl_step_actions_device(world.h, taken.data_ptr(), rewards.data_ptr(), dones.data_ptr()) == 0
        world.synchronize()
        lp, ent, stats = torch.empty(n, device="cuda"), torch.empty(n, device="cuda"), torch.empty(n, 4, device="cuda")
        best, best_lp = torch.empty(n, 1, dtype=torch.int32, device="cuda"), torch.empty(n, 1, device="cuda")
        rows = pkg.PolicyRows(logits.data_ptr(), pkg.F32, n, 4, taken=taken.data_ptr())
        pkg.policy_logprobs(rows, lp.data_ptr(), ent.data_ptr(), stats.data_ptr(), 1, best.data_ptr(), best_lp.data_ptr())
        advantage = rewards - rewards.mean()
        gl, gh = -advantage / n, torch.full((n,), -0.01 / n, device="cuda")
        grad = torch.empty_like(logits)
        pkg.policy_logprobs_backward(rows, stats.data_ptr(), gl.data_ptr(), gh.data_ptr(), grad.data_ptr())
        z = logits.double().requires_grad_()
        logp = torch.log_softmax(z, 1)
        e64 = -(logp.exp() * logp).sum(1)
        lp64 = logp.gather(1, taken.long()[:, None])[:, 0]
        (lp64 * gl + e64 * gh).sum().backward()
        assert (lp - lp64).abs().max() < 2e-6 and (ent - e64).abs().max() < 2e-6
        assert (grad - z.grad).abs().max() <= 2e-6 * (gl.abs().max() + gh.abs().max())
        assert torch.equal(best[:, 0].long(), (logits == logits.amax(1, keepdim=True)).int().argmax(1))
        keep[0].zero_().index_add_(0, cell, grad)
        keep[1].copy_(grad.sum(0))
        before = [p.double() for p in (table, bias)]
        opt.step(0.05)
        assert opt.get_stats().step == step + 1
        for p, b in zip((table, bias), before):
            assert torch.isfinite(p).all() and (p.double() - b).abs().max() <= 0.05 * 3.2      # |m / sqrt v| of a step is at most (1 - b1) / sqrt(1 - b2)
    s = opt.get_stats()
    want = torch.cat([k.reshape(-1) for k in keep]).double().norm()
    assert abs(s.grad_norm - float(want)) <= 1e-9 * float(want)


@pytest.mark.parametrize("max_norm", [0.0, 1.0])
def test_calls_after_a_refused_one(pkg, max_norm):
    """What failed and was reported -- an optimizer or a world on a device that is not there -- is not reported again by the next call, whose kernels it has nothing to do with."""
    net = Net(pkg, [3000, 50])
    opt = pkg.AdamW(net.list(), max_grad_norm=max_norm)
    nowhere = pkg.make_config(4, 4, 2, 1)
    nowhere.device = 1000
    x, lp, grad = (torch.randn(6, v, device="cuda") for v in (1500, 1, 1500))
    taken = torch.zeros(6, dtype=torch.int32, device="cuda")
    stats = torch.zeros(6, 4, device="cuda")

    def refused(first):
        if first:
            with pytest.raises(pkg.CudarlError):
                pkg.AdamW(net.list(), device=1000)
        else:
            with pytest.raises(pkg.CudarlError):
                pkg.VecGridWorld(nowhere)

    world = pkg.VecGridWorld(pkg.make_config(4, 4, 2, 1))
    for first in (True, False):
        before = net.snapshot()
        step = int(opt.get_stats().step) + 1
        refused(first)
        opt.step(0.01)
        norm = np.sqrt(sum((g ** 2).sum() for _w, g, _m, _v in before))
        check(net, before, step, 0.01, min(1.0, max_norm / (norm + 1e-6)) if max_norm else 1.0)
        for v in (7, 300, 1500):
            rows = pkg.PolicyRows(x.data_ptr(), pkg.F32, 6, v, row_stride=1500, taken=taken.data_ptr())
            refused(first)
            pkg.policy_logprobs(rows, lp.data_ptr(), stats=stats.data_ptr())
            refused(first)
            pkg.policy_logprobs_backward(rows, stats.data_ptr(), lp.data_ptr(), None, grad.data_ptr(), 1500)
    refused(True)
    world.train_steps(2)                                                     # the arena's own calls neither
    world.synchronize()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("max_norm", [0.0, 1.0])
def test_a_wait_that_runs_out(pkg, bits, max_norm):
    """The step gives up (its wait is for copies that nobody has begun), is not counted and is reported; no later step of the handle does anything; the GPU and a new
    handle go on."""
    net = Net(pkg, [300, 50000, 7], "bf16", "bf16", True, bits)
    opt = pkg.AdamW(net.list(), state_bits=bits, max_grad_norm=max_norm, step=4)
    opt.step(0.01)
    whole = [a.clone() for a, _o, _n in net.all]
    opt.debug_set_copy_wait_polls(3)
    opt.step(0.01)
    stats = pkg.AdamWStats()
    for _ in range(2):
        assert pkg.load().cudarl_adamw_get_stats(opt.h, C.byref(stats)) == 3000 + 32 and (stats.step, stats.skipped) == (5, 0)
        opt.debug_set_copy_wait_polls(0)
        opt.step(0.01)                                                       # launched as usual, and leaves everything as it is
    with pytest.raises(pkg.CudarlError, match="ran out"):
        opt.get_stats()
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, (b, _o, _n) in zip(whole, net.all))
    before = net.snapshot()
    norm = np.sqrt(sum((g ** 2).sum() for _w, g, _m, _v in before))
    opt = pkg.AdamW(net.list(), state_bits=bits, max_grad_norm=max_norm, step=5)
    opt.step(0.01)
    check(net, before, 6, 0.01, min(1.0, max_norm / (norm + 1e-6)) if max_norm else 1.0)
    assert opt.get_stats().step == 6
    with pytest.raises(pkg.CudarlError, match="polls"):
        opt.debug_set_copy_wait_polls(-1)


@pytest.mark.parametrize("bits", [32, 8])
def test_the_weights_of_a_policy_that_steps_the_arena(pkg, bits):
    """A policy (a table of logits over the cells, a shared bias) chooses the moves, the calls give its gradient, and its weights and moments after every step are those of
    the formula in 64 bits, from the weights, moments and gradients before it."""
    w, h, n = 12, 9, 500
    world = pkg.VecGridWorld(pkg.make_config(w, h, n, 99, obstacle_kind=pkg.OBST_BERNOULLI, obstacle_p=0.1, goal_mode=pkg.GOAL_SEEDED, num_goals=1, start_mode=pkg.START_RANDOM))
    gen = torch.Generator("cuda").manual_seed(1)
    net = Net(pkg, [w * h * 4, 4], bits=bits)
    for t in net.tensors:
        for key in ("m", "v", "s1", "s2"):
            if key in t:
                t[key].zero_()
    table, bias = net.tensors[0]["param"].view(w * h, 4), net.tensors[1]["param"]
    opt = pkg.AdamW(net.list(), state_bits=bits, max_grad_norm=0.002, seed=12)
    rewards, dones = torch.zeros(n, device="cuda"), torch.zeros(n, dtype=torch.uint8, device="cuda")
    clipped = 0
    for step in range(1, 7):
        x, y, _t = world.get_state()
        cell = torch.from_numpy(y.astype(np.int64) * w + x).cuda()
        logits = (table[cell] + bias).contiguous()
        noise = -torch.log(-torch.log(torch.rand(n, 4, device="cuda", generator=gen).clamp(1e-6, 1 - 1e-6)))
        taken = (logits + noise).argmax(1).int()
        torch.cuda.synchronize()
        assert pkg.load().cudarl_step_actions_device(world.h, taken.data_ptr(), rewards.data_ptr(), dones.data_ptr()) == 0
        world.synchronize()
        rows = pkg.PolicyRows(logits.data_ptr(), pkg.F32, n, 4, taken=taken.data_ptr())
        lp, grad = torch.empty(n, device="cuda"), torch.empty_like(logits)
        pkg.policy_logprobs(rows, lp.data_ptr())
        gl, gh = -(rewards - rewards.mean()) / n, torch.full((n,), -0.01 / n, device="cuda")
        pkg.policy_logprobs_backward(rows, None, gl.data_ptr(), gh.data_ptr(), grad.data_ptr())
        net.tensors[0]["grad"].view(w * h, 4).zero_().index_add_(0, cell, grad)
        net.tensors[1]["grad"].copy_(grad.sum(0))
        before = net.snapshot()
        norm = np.sqrt(sum((g ** 2).sum() for _w, g, _m, _v in before))
        clipped += norm > 0.002
        opt.step(0.05)
        check(net, before, step, 0.05, min(1.0, float(np.float32(0.002)) / (norm + 1e-6)), seed=12)
        assert any((t["param"].double().cpu().numpy() != b[0]).any() for t, b in zip(net.tensors, before))
    assert clipped > 0


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("beta1,beta2,step", [(0.0, 0.0, 0), (0.0, 0.999, 3), (0.9, 0.0, 0), (0.999999, 1 - 1e-9, 0), (0.9, 0.999, 10 ** 15), (0.5, 0.999999, 1 << 62)])
def test_settings_at_their_ends(pkg, bits, beta1, beta2, step):
    net = Net(pkg, [300, 5000, 1], "f32", "bf16", False, bits, seed=4)
    before = net.snapshot()
    opt = pkg.AdamW(net.list(), state_bits=bits, beta1=beta1, beta2=beta2, seed=2, step=step)
    opt.step(0.01)
    check(net, before, step + 1, 0.01, 1.0, 2, beta1, beta2)
    assert opt.get_stats().step == step + 1
    before = net.snapshot()
    opt.step(0.0, grad_scale=0.5)                                            # moments move, weights do not
    for t, (_w, g, m, v) in zip(net.tensors, before):
        # the two terms of m' may cancel -- all of a tensor of one value: it is off by three roundings of the terms, whatever is left of them
        off = 4 * U * (beta1 * np.abs(m) + (1 - beta1) * np.abs(0.5 * g)) + 1e-37
        em, ev = beta1 * m + (1 - beta1) * 0.5 * g, beta2 * v + (1 - beta2) * 0.25 * g * g
        if bits == 32:
            assert (np.abs(t["m"].double().cpu().numpy() - em) <= off).all() and (np.abs(t["v"].double().cpu().numpy() - ev) <= 5 * U * ev + 1e-37).all()
            continue
        value = np.concatenate([plain.E4M3, [np.nan], -plain.E4M3, [np.nan]])
        blocks = [slice(b, b + 256) for b in range(0, len(g), 256)]
        for key, scale, x, o in (("m", "s1", em, off), ("v", "s2", np.sqrt(ev), 3 * U * np.sqrt(ev))):
            got, by = t[key].cpu().numpy(), t[scale].double().cpu().numpy()
            for b, at in enumerate(blocks):
                high = np.abs(x[at]).max() / 448
                assert abs(by[b] - high) <= 4 * U * high + o[at].max() / 448
                assert (np.abs(value[got[at]] * by[b] - x[at]) <= np.maximum(np.abs(x[at]) / 8, by[b] * 2.0 ** -9) * (1 + 8 * U) + o[at]).all()
    assert all((t["param"].double().cpu().numpy() == b[0]).all() for t, b in zip(net.tensors, before))


@pytest.mark.parametrize("bits", [32, 8])
def test_a_tensor_beyond_32_bits(pkg, bits):
    """2^31 + 777 values: pieces of it on both sides of every power of two, its end, and the rest left at zero."""
    n = (1 << 31) + 777
    param, grad = torch.zeros(n, dtype=torch.bfloat16, device="cuda"), torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    m, v = (torch.zeros(n, dtype=torch.float32 if bits == 32 else torch.uint8, device="cuda") for _ in range(2))
    s1, s2 = (torch.zeros((n + 255) // 256, device="cuda") for _ in range(2))
    windows = [0, (1 << 28) - 256, (1 << 29) - 256, (1 << 30) - 256, (1 << 31) - 512, (1 << 31), n - 521]
    windows = [w - w % 256 for w in windows]
    gen = torch.Generator("cuda").manual_seed(1)
    for w in windows:
        for x, size in ((param, 1.0), (grad, 1e-2)):                         # (a window may reach into the next)
            x[w:w + 512] = (torch.randn(min(512, n - w), device="cuda", generator=gen) * size).bfloat16()
    tensors = [pkg.AdamWTensor(count=n, param=param.data_ptr(), param_type=pkg.BF16, grad=grad.data_ptr(), grad_type=pkg.BF16, moment1=m.data_ptr(), moment2=v.data_ptr(),
                               scale1=s1.data_ptr(), scale2=s2.data_ptr(), lr_scale=1.0, weight_decay=0.01)]
    before = [(param[w:w + 512].double().cpu().numpy(), grad[w:w + 512].double().cpu().numpy()) for w in windows]
    total = sum(float(part.double().square().sum()) for part in grad.split(1 << 28))
    opt = pkg.AdamW(tensors, state_bits=bits, max_grad_norm=0.1, seed=9)
    opt.step(0.01)
    norm = np.sqrt(total)
    assert abs(opt.get_stats().grad_norm - norm) <= 1e-12 * norm
    clip = min(1.0, float(np.float32(0.1)) / (norm + 1e-6))
    for w, (p, g) in zip(windows, before):
        ep, em, ev = plain.adamw(p, g, np.zeros_like(p), np.zeros_like(p), 1, float(np.float32(0.01)), float(np.float32(0.01)), clip)
        assert (np.abs(param[w:w + 512].double().cpu().numpy() - ep) <= 1e-6 * 0.01 + plain.HALF_STEP["bf16"] * np.abs(ep) * (1 + 2.0 ** -7)).all()
        for x, scale, want in ((m, s1, em), (v, s2, np.sqrt(ev))):
            if bits == 32:
                want = want if x is m else ev
                assert (np.abs(x[w:w + 512].double().cpu().numpy() - want) <= 6 * U * np.abs(want) + 1e-37).all()
            else:
                value = np.concatenate([plain.E4M3, [np.nan], -plain.E4M3, [np.nan]])
                by = scale[w // 256:w // 256 + 2].double().cpu().numpy().repeat(256)[:len(want)]
                got = value[x[w:w + 512].cpu().numpy()] * by
                assert (np.abs(got - want) <= np.maximum(np.abs(want) / 8, by * 2.0 ** -9) * 1.001).all()
    for w in windows:                                                        # elsewhere nothing has become anything
        for x in (param, m, v):
            x[w:w + 512] = 0
    assert not any(bool(part.any()) for x in (param, m, v) for part in x.split(1 << 28))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("offset", [0, 1, 4])
def test_new_gradients_for_a_captured_step(pkg, bits, offset):
    """A captured step reads the gradients where they are when it is replayed, aligned as they are then."""
    net = Net(pkg, [3000, 0, 50], bits=bits)
    opt = pkg.AdamW(net.list(), state_bits=bits, max_grad_norm=0.5)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        opt.step(0.01, stream=torch.cuda.current_stream().cuda_stream)
    for step in (1, 2):
        grads = [torch.randn(n + offset, device="cuda")[offset:] for n in net.sizes]
        opt.set_gradients([x.data_ptr() if x.numel() else None for x in grads])
        before = [(w, x.double().cpu().numpy(), m, v) for (w, _g, m, v), x in zip(net.snapshot(), grads)]
        norm = np.sqrt(sum((x ** 2).sum() for _w, x, _m, _v in before))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        check(net, before, step, 0.01, 0.5 / (norm + 1e-6))
    del g


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("bad", [np.inf, np.nan])
def test_a_gradient_that_is_no_number_without_clipping(pkg, bits, bad):
    """Its weight becomes NaN; every other takes its step, and outside its block goes on."""
    net = Net(pkg, [300, 5000], bits=bits)
    net.tensors[1]["grad"][1025] = bad
    before = net.snapshot()
    opt = pkg.AdamW(net.list(), state_bits=bits)
    opt.step(0.01)
    weight = net.tensors[1]["param"].double().cpu().numpy()
    w, g, m, v = before[1]
    g = g.copy(); g[1025] = 0.0
    ew, _m, _v = plain.adamw(w, g, m, v, 1, float(np.float32(0.01)), float(np.float32(net.decay)), lr_scale=1.5)
    keep = np.arange(5000) != 1025
    assert np.isnan(weight[1025]) and np.isfinite(weight[keep]).all()
    assert (np.abs(weight - ew)[keep] <= 1e-6 * np.maximum(1, np.abs(ew - w)[keep]) + 2 * U * np.abs(ew)[keep]).all()
    opt.step(0.01)
    after = net.tensors[1]["param"].double().cpu().numpy()
    outside = (np.arange(5000) < 1024) | (np.arange(5000) >= 1280)
    assert np.isfinite(after[outside]).all() and (after[outside] != weight[outside]).any()
