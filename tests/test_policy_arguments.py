"""The learned policy's entry points refuse what they cannot do, before anything is launched: no GPU is needed to be refused."""
import ctypes as C

import pytest

A = 1 << 20                                                   # an address that is aligned to everything and never read


def rows(pkg, **kw):
    return pkg.PolicyRows(**{**dict(logits=A, type=pkg.F32, rows=3, actions=5, taken=A), **kw})


def text(pkg):
    return pkg.load().cudarl_last_global_error().decode()


def test_struct_sizes(pkg):
    assert pkg.MAX_TOP == 32 and pkg.ADAMW_BLOCK == 256
    assert [C.sizeof(t) for t in (pkg.PolicyRows, pkg.AdamWTensor, pkg.AdamWConfig, pkg.AdamWStats)] == [72, 80, 56, 24]


@pytest.mark.parametrize("kw,word", [
    (dict(struct_size=8), "struct_size"), (dict(type=3), "type"), (dict(type=-1), "type"), (dict(rows=-1), "rows"), (dict(actions=0), "actions"), (dict(actions=1 << 31), "actions"),
    (dict(row_stride=4), "row_stride"), (dict(row_stride=1 << 60), "strides"), (dict(rows=1 << 38, row_stride=1 << 38), "strides"), (dict(legal=A, legal_stride=4), "legal_stride"), (dict(legal=A, legal_stride=-1), "legal_stride"),
    (dict(actions=(1 << 30) + 1), "actions"), (dict(inv_temperature=0.0), "inv_temperature"), (dict(inv_temperature=9e-7), "inv_temperature"), (dict(inv_temperature=2e6), "inv_temperature"), (dict(inv_temperature=-1.0), "inv_temperature"), (dict(inv_temperature=float("inf")), "inv_temperature"),
    (dict(inv_temperature=float("nan")), "inv_temperature"), (dict(logits=None), "logits"), (dict(logits=A + 2), "aligned")])
def test_rows_are_refused(pkg, kw, word):
    lib = pkg.load()
    size = kw.pop("struct_size", None)
    p = rows(pkg, **kw)
    if size is not None:
        p.struct_size = size
    assert lib.cudarl_policy_logprobs(p, A, A, None, 0, None, None, None) == -1 and word in text(pkg)
    assert lib.cudarl_policy_logprobs_backward(p, A, A, A, A, max(1, p.actions), None) == -1 and word in text(pkg)


def test_outputs_are_refused(pkg):
    lib = pkg.load()
    assert lib.cudarl_policy_logprobs(None, A, A, None, 0, None, None, None) == -1
    assert lib.cudarl_policy_logprobs(rows(pkg), None, None, None, 0, None, None, None) == -1 and "no output" in text(pkg)
    assert lib.cudarl_policy_logprobs(rows(pkg, taken=None), A, None, None, 0, None, None, None) == -1 and "taken" in text(pkg)
    for top in (-1, pkg.MAX_TOP + 1):
        assert lib.cudarl_policy_logprobs(rows(pkg), A, A, None, top, A, A, None) == -1 and "top" in text(pkg)
    assert lib.cudarl_policy_logprobs(rows(pkg), A, A, None, 2, A, None, None) == -1 and "top" in text(pkg)
    assert lib.cudarl_policy_logprobs(rows(pkg, rows=0, logits=None, taken=None), None, None, None, 0, None, None, None) == 0


def test_gradients_are_refused(pkg):
    lib = pkg.load()
    b = lib.cudarl_policy_logprobs_backward
    assert b(None, A, A, A, A, 5, None) == -1
    assert b(rows(pkg), None, A, A, A, 5, None) == -1 and "stats" in text(pkg)
    assert b(rows(pkg), A, A, A, None, 5, None) == -1 and "grad_logits" in text(pkg)
    assert b(rows(pkg), A, A, A, A, 4, None) == -1 and "grad_stride" in text(pkg)
    assert b(rows(pkg), A, A, A, A, 1 << 60, None) == -1 and "grad_stride" in text(pkg)
    assert b(rows(pkg, taken=None), A, A, A, 2 * A, 5, None) == -1 and "taken" in text(pkg)
    assert b(rows(pkg, row_stride=6), A, A, A, A, 5, None) == -1 and "stride" in text(pkg)      # in place, but at another stride
    assert b(rows(pkg, rows=0), A, A, A, A, 5, None) == 0


def config(pkg, **kw):
    d = {**dict(struct_size=C.sizeof(pkg.AdamWConfig), device=0, state_bits=32, max_grad_norm=0.0, beta1=0.9, beta2=0.999, eps=1e-8, seed=0, step=0), **kw}
    return pkg.AdamWConfig(**d)


@pytest.mark.parametrize("kw,word", [(dict(struct_size=4), "struct_size"), (dict(device=-1), "device"), (dict(state_bits=16), "state_bits"), (dict(beta1=1.0), "beta1"), (dict(beta2=-0.1), "beta2"),
                                     (dict(beta1=float("nan")), "beta1"), (dict(eps=0.0), "eps"), (dict(eps=float("inf")), "eps"), (dict(max_grad_norm=-1.0), "max_grad_norm"),
                                     (dict(max_grad_norm=float("nan")), "max_grad_norm"), (dict(step=-1), "step")])
def test_configs_are_refused(pkg, kw, word):
    lib, h = pkg.load(), C.c_void_p()
    assert lib.cudarl_adamw_create(C.byref(config(pkg, **kw)), 0, None, C.byref(h)) == -1 and word in text(pkg) and not h.value


def test_null_arguments_are_refused(pkg):
    lib, h = pkg.load(), C.c_void_p()
    s = pkg.AdamWStats()
    assert lib.cudarl_adamw_create(None, 0, None, C.byref(h)) == -1
    assert lib.cudarl_adamw_create(C.byref(config(pkg)), 0, None, None) == -1
    assert lib.cudarl_adamw_create(C.byref(config(pkg)), 1, None, C.byref(h)) == -1
    assert lib.cudarl_adamw_create(C.byref(config(pkg)), -1, None, C.byref(h)) == -1
    assert lib.cudarl_adamw_step(None, 0.1, 1.0, None) == -1
    assert lib.cudarl_adamw_set_gradients(None, None, None) == -1
    assert lib.cudarl_adamw_get_stats(None, C.byref(s)) == -1
    lib.cudarl_adamw_destroy(None)


def test_the_debug_call_is_refused(pkg):
    assert pkg.load().cudarl_debug_adamw_set_copy_wait_polls(None, 1) == -1 and "null" in text(pkg)


def test_short_rows_need_no_statistics(pkg):
    """The gradient of rows of up to 128 actions takes the sums anew: there None is fine (what is refused here is the address of the logits), above not."""
    assert pkg.ACTIONS_WITHOUT_STATS == 128
    for actions, word in ((1, None), (128, None), (129, "stats"), (5000, "stats")):
        with pytest.raises(pkg.CudarlError) as e:
            pkg.policy_logprobs_backward(rows(pkg, actions=actions), None, A, A, A)
        assert ("stats" in str(e.value)) == (word is not None)
