"""Performance cases of the learned policy's operators: what a user trains a policy with that is no table.

Three kinds of use, through the entry points on the caller's own device arrays:

  evaluate   rows of logits -> log probability of the action taken, entropy, and the most probable actions;
  learn      the same with the statistics kept, then the gradient of a loss of the log probability and the entropy with respect to
             the logits -- the two calls of a policy-gradient step;
  adamw      one AdamW step over all tensors of a network, moments in 32 bits or in 8, with or without clipping by the global norm.

Where `own` is false the operators are computed in their plain form.  Moments of 8 bits are e4m3 codes with one scale for 256 values; the
code is rounded up or down at random, by 16 bits of the Philox stream of (seed, step, place).
"""
import importlib.util
import math
import os
import random
import sys

import torch

own = False

TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
INF = float("inf")
BLOCK = 256                    # values of one scale
E4M3_MAX = 448.0
BETA1, BETA2, EPS, LR = 0.9, 0.999, 1e-8, 1e-4
OPTIMIZER_TAG = 0x4F50544D


def _package():
    name = "cudarl_arena_b200"
    if name not in sys.modules:
        here = os.path.join(os.getcwd(), "cudarl-arena_b200")
        spec = importlib.util.spec_from_file_location(name, os.path.join(here, "__init__.py"), submodule_search_locations=[here])
        sys.modules[name] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules[name])
    return sys.modules[name]


def listed():
    return [
        # The small arena's environments choose among their four moves: what a rollout calls every step, launch latency.
        dict(name="evaluate_4096x4", kind="evaluate", type="f32", rows=4096, actions=4, top=1, mask=False, pad=0, temperature=1.0),
        # The medium arena with joint actions, rows with a stride of their own, illegal actions masked, a sampling temperature.
        dict(name="evaluate_65536x257_masked", kind="evaluate", type="f32", rows=65536, actions=257, top=4, mask=True, pad=7, temperature=0.7),
        # One step of decoding for one sequence of a language-model policy.
        dict(name="evaluate_1x131072", kind="evaluate", type="bf16", rows=1, actions=131072, top=20, mask=False, pad=0, temperature=1.0),
        # A few hundred sequences with constrained choices, an odd vocabulary.
        dict(name="evaluate_500x50001_masked", kind="evaluate", type="f16", rows=500, actions=50001, top=8, mask=True, pad=0, temperature=0.8),
        # Scoring a batch of long answers.
        dict(name="evaluate_4096x131072", kind="evaluate", type="bf16", rows=4096, actions=131072, top=5, mask=False, pad=0, temperature=1.0),
        # The headline arena: 4.2 million environments with four moves each.
        dict(name="learn_4194304x4", kind="learn", type="f32", rows=4194304, actions=4, top=0, mask=False, pad=0, temperature=1.0),
        # A minibatch of a macro-action policy, masked.
        dict(name="learn_4001x1001_masked", kind="learn", type="bf16", rows=4001, actions=1001, top=0, mask=True, pad=0, temperature=1.0),
        # A training batch of a language-model policy with an odd vocabulary: rows begin at every alignment.
        dict(name="learn_2047x65537", kind="learn", type="bf16", rows=2047, actions=65537, top=0, mask=False, pad=0, temperature=1.0),
        # A small policy network: latency.
        dict(name="adamw_100k_f32", kind="adamw", params=100_000, tensors=8, param="f32", master=False, grad="f32", bits=32, clip=True),
        # Many odd tensors, gradients in half precision, moments of 8 bits, clipped.
        dict(name="adamw_9m_8bit_ragged", kind="adamw", params=9_000_001, tensors=777, param="f32", master=False, grad="f16", bits=8, clip=True),
        # A network in mixed precision: weights and gradients in bf16, the weights' masters and the moments in fp32.
        dict(name="adamw_150m_mixed", kind="adamw", params=150_000_000, tensors=150, param="bf16", master=True, grad="bf16", bits=32, clip=False),
        # The same with moments of 8 bits, clipped: what lets a larger network train beside the arena's own tables.
        dict(name="adamw_200m_8bit", kind="adamw", params=200_000_000, tensors=200, param="bf16", master=True, grad="bf16", bits=8, clip=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["evaluate", "learn", "adamw"])
    if kind == "adamw":
        params = _log(rng, 5_000, 100_000_000)
        param = rng.choice(["f32", "bf16", "f16"])
        return dict(kind=kind, params=params, tensors=min(_log(rng, 1, 600), 1 + params // 2000), param=param, master=param != "f32" and rng.random() < 0.7,
                    grad=rng.choice(["f32", "bf16", "f16"]), bits=rng.choice([8, 32]), clip=rng.random() < 0.5)
    actions = _log(rng, 2, 200_000)
    rows = min(_log(rng, 1, 2_000_000), max(1, 100_000_000 // actions))
    return dict(kind=kind, type=rng.choice(["f32", "bf16", "f16"]), rows=rows, actions=actions, top=min(actions, rng.choice([0, 1, 3, 20, 32])) if kind == "evaluate" else 0,
                mask=rng.random() < 0.3, pad=rng.choice([0, 0, 1, 6]), temperature=rng.choice([1.0, 1.0, 0.6, 1.3]))


def _sizes(case):
    """The tensors' lengths: a few large ones and many small, odd ones among them; they go by the case alone."""
    rng = random.Random(case["params"] * 31 + case["tensors"])
    weight = [math.exp(rng.gauss(0, 2)) for _ in range(case["tensors"])]
    return [max(1, int(case["params"] * w / sum(weight))) for w in weight]


def _blocks(n):
    return (n + BLOCK - 1) // BLOCK


# ---------------------------------------------------------------------------------------------------------------- inputs


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    def rand(*shape):
        return torch.rand(*shape, generator=gen, device="cuda")

    if case["kind"] == "adamw":
        return _prepare_adamw(case, seed, randn, rand)
    n, v = case["rows"], case["actions"]
    logits = torch.empty(n, v + case["pad"], dtype=TORCH[case["type"]], device="cuda")
    part = max(1, (1 << 27) // (v + case["pad"]))
    for at in range(0, n, part):
        rows = min(part, n - at)
        logits[at:at + rows] = randn(rows, v + case["pad"]) * (0.5 + 3.0 * rand(rows, 1)) + 2.0 * randn(rows, 1)
    state = dict(case=case, logits=logits[:, :v])
    taken = (rand(n).double() * v).to(torch.int32).clamp_(0, v - 1)
    if case["mask"]:
        legal = rand(n, v) < 0.7
        legal.scatter_(1, taken.long()[:, None], True)                       # the action that was taken was a legal one
        legal[torch.arange(n, device="cuda") % 97 == 96] = False             # environments that are done have nothing left to choose
        state["legal"] = legal.to(torch.uint8)
    taken[torch.arange(n, device="cuda") % 101 == 100] = -1                  # padding of a batch of sequences
    state["taken"] = taken
    if case["kind"] == "learn":
        state["grad_logprob"] = -randn(n)                                    # advantages
        state["grad_entropy"] = torch.full((n,), -0.01, device="cuda")
    return state


def _prepare_adamw(case, seed, randn, rand):
    """A network's tensors in flat buffers, each tensor at a multiple of 256 values; between them there are zeros."""
    sizes = _sizes(case)
    blocks = [_blocks(n) for n in sizes]
    total = sum(blocks) * BLOCK
    of_block = torch.repeat_interleave(torch.arange(len(sizes)), torch.tensor(blocks)).cuda()
    length = torch.tensor(sizes).cuda()[of_block]
    first = (torch.cumsum(torch.tensor(blocks), 0) - torch.tensor(blocks)).cuda()[of_block]
    place = (torch.arange(len(of_block), device="cuda") - first)[:, None] * BLOCK + torch.arange(BLOCK, device="cuda")
    used = (place < length[:, None]).reshape(-1)
    size = torch.exp(1.5 * randn(len(sizes)))[of_block][:, None].expand(-1, BLOCK).reshape(-1)     # every tensor's gradients have a size of their own
    p = randn(total) * 0.1 * used
    grad = randn(total) * 2e-3 * size * used
    m = randn(total) * 5e-4 * size * used
    root = (0.5 + rand(total)) * 2e-3 * size * used
    del place, size
    state = dict(case=case, seed=seed, t=100, sizes=sizes, of_block=of_block, decay=[0.01 if n > 4096 else 0.0 for n in sizes])
    state["decays"] = torch.tensor(state["decay"], device="cuda")
    state["grad"] = grad.to(TORCH[case["grad"]])
    state["param"] = p.to(TORCH[case["param"]])
    if case["master"]:
        state["master"] = p
    if case["bits"] == 32:
        state["m"], state["v"] = m, root * root
    else:
        for key, x in (("m", m), ("v", root)):
            scale = x.reshape(-1, BLOCK).abs().amax(1) / E4M3_MAX
            state[key] = (x.reshape(-1, BLOCK) / scale.clamp_min(1e-30)[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).reshape(-1)
            state[key + "_scale"] = scale
    del p, grad, m, root, used
    if own:                                                                  # the optimizer's handle, made once for a network
        pkg = _package()
        types = {"f32": pkg.F32, "bf16": pkg.BF16, "f16": pkg.F16}
        tensors, at = [], 0
        for n, decay in zip(sizes, state["decay"]):
            def pointer(key, per=1):
                return state[key][at // per:].data_ptr() if key in state else None
            tensors.append(pkg.AdamWTensor(count=n, param=pointer("param"), param_type=types[case["param"]], grad=pointer("grad"), grad_type=types[case["grad"]],
                                           master=pointer("master"), moment1=pointer("m"), moment2=pointer("v"), scale1=pointer("m_scale", BLOCK), scale2=pointer("v_scale", BLOCK),
                                           lr_scale=1.0, weight_decay=decay))
            at += _blocks(n) * BLOCK
        state["optimizer"] = pkg.AdamW(tensors, state_bits=case["bits"], beta1=BETA1, beta2=BETA2, eps=EPS, max_grad_norm=1.0 if case["clip"] else 0.0, seed=seed, step=state["t"])
    return state


# ---------------------------------------------------------------------------------------------------------------- one pass


def run(state):
    kind = state["case"]["kind"]
    if kind == "adamw":
        return _run_adamw(state)
    if own:
        return _run_policy(state)
    return _plain_evaluate(state) if kind == "evaluate" else _plain_learn(state)


def _run_policy(state):
    pkg, case = _package(), state["case"]
    logits, n, top = state["logits"], case["rows"], case["top"]
    stream = torch.cuda.current_stream().cuda_stream
    legal = state.get("legal")
    rows = pkg.PolicyRows(logits=logits.data_ptr(), type={"f32": pkg.F32, "bf16": pkg.BF16, "f16": pkg.F16}[case["type"]], rows=n, actions=case["actions"],
                          row_stride=logits.stride(0), legal=legal.data_ptr() if legal is not None else None, legal_stride=legal.stride(0) if legal is not None else 0,
                          taken=state["taken"].data_ptr(), inv_temperature=1.0 / case["temperature"])
    logprob, entropy = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    out = dict(logprob=logprob, entropy=entropy)
    if case["kind"] == "evaluate":
        if top:
            out["top_actions"], out["top_logprobs"] = torch.empty(n, top, dtype=torch.int32, device="cuda"), torch.empty(n, top, device="cuda")
            pkg.policy_logprobs(rows, logprob.data_ptr(), entropy.data_ptr(), top=top, top_actions=out["top_actions"].data_ptr(), top_logprobs=out["top_logprobs"].data_ptr(),
                                stream=stream)
        else:
            pkg.policy_logprobs(rows, logprob.data_ptr(), entropy.data_ptr(), stream=stream)
        return out
    stats = torch.empty(n, 4, device="cuda")
    grad = torch.empty(n, case["actions"], dtype=logits.dtype, device="cuda")
    pkg.policy_logprobs(rows, logprob.data_ptr(), entropy.data_ptr(), stats=stats.data_ptr(), stream=stream)
    pkg.policy_logprobs_backward(rows, stats.data_ptr(), state["grad_logprob"].data_ptr(), state["grad_entropy"].data_ptr(), grad.data_ptr(), case["actions"], stream=stream)
    out["grad"] = grad
    return out


def _plain_rows(state):
    """d = (x - max) / temperature, log sum e^d, entropy, log probability of the action taken."""
    case = state["case"]
    x = state["logits"].float()
    if "legal" in state:
        x = x.masked_fill(state["legal"] == 0, -INF)
    high = x.amax(1, keepdim=True)
    none = high == -INF
    d = (x - high.masked_fill(none, 0.0)) * (1.0 / case["temperature"])
    e = d.exp()
    total = e.sum(1)
    log_total = total.log()
    entropy = log_total - torch.where(e > 0, d * e, 0.0).sum(1) / total
    entropy = entropy.masked_fill(none[:, 0], 0.0)
    taken = state["taken"].long()
    was = (taken >= 0) & (taken < case["actions"])
    logprob = d.gather(1, taken.clamp(0, case["actions"] - 1)[:, None])[:, 0] - log_total
    logprob = torch.where(was, logprob.masked_fill(none[:, 0], -INF), 0.0)
    return x, d, e, total, log_total, entropy, logprob, none, taken, was


def _plain_evaluate(state):
    x, d, _e, _total, log_total, entropy, logprob, none, _taken, _was = _plain_rows(state)
    out = dict(logprob=logprob, entropy=entropy)
    top, v = state["case"]["top"], state["case"]["actions"]
    if top:
        bits = (x + 0.0).view(torch.int32)
        bits = bits ^ ((bits >> 31) & 0x7FFFFFFF)                            # integers in the order of the values
        key = bits.long() * (1 << 32) + (v - 1 - torch.arange(v, device="cuda"))
        at = (v - 1) - (key.topk(top, dim=1).values & 0xFFFFFFFF)
        there = x.gather(1, at) > -INF
        out["top_actions"] = torch.where(there, at, -1).to(torch.int32)
        out["top_logprobs"] = torch.where(there, d.gather(1, at) - log_total[:, None], -INF)
    return out


def _plain_learn(state):
    _x, d, e, total, log_total, entropy, logprob, none, taken, was = _plain_rows(state)
    case = state["case"]
    gl = torch.where(was, state["grad_logprob"], 0.0)[:, None]
    gh = state["grad_entropy"][:, None]
    p = e / total[:, None]
    log_p = (d - log_total[:, None]).clamp_min(-1e30)
    grad = -p * (gl + gh * (log_p + entropy[:, None]))
    grad.scatter_add_(1, taken.clamp(0, case["actions"] - 1)[:, None], gl)
    grad = (grad * (1.0 / case["temperature"])).masked_fill(none, 0.0)
    if "legal" in state:
        grad = grad.masked_fill(state["legal"] == 0, 0.0)
    return dict(logprob=logprob, entropy=entropy, grad=grad.to(state["logits"].dtype))


def _philox(quads, step, seed):
    """Philox4x32-10 of the counters (quad, step) under the key of the seed: four words of 32 bits for every quad."""
    low = 0xFFFFFFFF
    c = [quads & low, quads >> 32, torch.full_like(quads, step & low), torch.full_like(quads, step >> 32)]
    k = [seed & low, ((seed >> 32) & low) ^ OPTIMIZER_TAG]

    def wide(a, b):                                                          # 32 x 32 -> two words; the product itself would pass 63 bits
        lo = (a & 0xFFFF) * b
        hi = (a >> 16) * b + (lo >> 16)
        return hi >> 16, ((hi << 16) | (lo & 0xFFFF)) & low

    for _ in range(10):
        hi0, lo0 = wide(c[0], 0xD2511F53)
        hi1, lo1 = wide(c[2], 0xCD9E8D57)
        c = [hi1 ^ c[1] ^ k[0], lo1, hi0 ^ c[3] ^ k[1], lo0]
        k = [(k[0] + 0x9E3779B9) & low, (k[1] + 0xBB67AE85) & low]
    return torch.stack(c, 1).reshape(-1)


def _to_codes(x, bits16, up_from_zero):
    """x, 256 values a row, as e4m3 codes and scales: rounded up or down by 16 random bits each."""
    scale = x.abs().amax(1) / E4M3_MAX
    y = (x.abs() / torch.where(scale > 0, scale, 1.0)[:, None]).clamp_max(E4M3_MAX)
    small = y < 2.0 ** -6                                                    # below the smallest normal code the steps are all alike
    z = torch.where(small, y + 2.0 ** -6, y)
    code = ((z.view(torch.int32) + (bits16 << 4).to(torch.int32)) >> 20) - torch.where(small, 121 << 3, 120 << 3)
    if up_from_zero:
        code = torch.where((x > 0) & (code == 0), 1, code)
    code = code | torch.where(x < 0, 128, 0)
    return code.to(torch.uint8).view(torch.float8_e4m3fn).reshape(-1), scale


def _run_adamw(state):
    case = state["case"]
    if own:
        state["optimizer"].step(LR, stream=torch.cuda.current_stream().cuda_stream)
    else:
        _plain_adamw(state)
    return {key: state[key] for key in ("param", "master", "m", "v", "m_scale", "v_scale") if key in state}


def _plain_adamw(state):
    case = state["case"]
    state["t"] += 1
    t = state["t"]
    g = state["grad"].float().reshape(-1, BLOCK)
    if case["clip"]:
        norm = state["grad"].double().square().sum().sqrt()
        g = g * (1.0 / (norm + 1e-6)).clamp_max(1.0).float()
    if case["bits"] == 32:
        m, v = state["m"].reshape(-1, BLOCK), state["v"].reshape(-1, BLOCK)
    else:
        m = state["m"].float().reshape(-1, BLOCK) * state["m_scale"][:, None]
        v = (state["v"].float().reshape(-1, BLOCK) * state["v_scale"][:, None]).square()
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * g * g
    p = (state["master"] if case["master"] else state["param"].float()).reshape(-1, BLOCK)
    step = (m / (1 - BETA1 ** t)) / ((v / (1 - BETA2 ** t)).sqrt() + EPS)
    p = p - LR * (state["decays"][state["of_block"]][:, None] * p + step)
    if case["master"]:
        state["master"].copy_(p.reshape(-1))
    state["param"].copy_(p.reshape(-1))
    if case["bits"] == 32:
        state["m"].copy_(m.reshape(-1))
        state["v"].copy_(v.reshape(-1))
    else:
        words = _philox(torch.arange(g.numel() // 4, device="cuda"), t, state["seed"]).reshape(-1, BLOCK)
        for key, x, bits16 in (("m", m, words & 0xFFFF), ("v", v.sqrt(), words >> 16)):
            code, scale = _to_codes(x, bits16, key == "v")
            state[key].copy_(code)
            state[key + "_scale"].copy_(scale)


# ---------------------------------------------------------------------------------------------------------------- work and exact values


def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2}
    if case["kind"] == "adamw":
        n = sum(_sizes(case))
        moments = 8.0 if case["bits"] == 32 else 2.0 + 8.0 / BLOCK
        weights = size[case["param"]] * (1 if case["master"] else 2) + (8 if case["master"] else 0)      # with a master the weights are written only
        return dict(bytes=n * (size[case["grad"]] + weights + 2 * moments), flops=n * (20 if case["bits"] == 32 else 60))
    cells = case["rows"] * case["actions"]
    read = cells * (size[case["type"]] + (1 if case["mask"] else 0))
    if case["kind"] == "evaluate":
        return dict(bytes=read + case["rows"] * (12 + 8 * case["top"]), flops=5 * cells)
    return dict(bytes=read + cells * size[case["type"]] + case["rows"] * 20, flops=13 * cells)       # the logits in once, the gradient out


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "adamw":
        return _exact_adamw(state)
    n, v, top = case["rows"], case["actions"], case["top"]
    out = dict(logprob=torch.empty(n, dtype=torch.float64, device="cuda"), entropy=torch.empty(n, dtype=torch.float64, device="cuda"))
    if top:
        out["top_actions"], out["top_logprobs"] = None, torch.empty(n, top, dtype=torch.float64, device="cuda")
    if case["kind"] == "learn":
        out["grad"] = torch.empty(n, v, dtype=torch.float64, device="cuda")
    part = max(1, (1 << 26) // v)
    for at in range(0, n, part):
        rows = slice(at, min(n, at + part))
        z = state["logits"][rows].double() / case["temperature"]
        if "legal" in state:
            z[state["legal"][rows] == 0] = -INF
        logp = z - torch.logsumexp(z, 1, keepdim=True)
        empty = torch.isinf(z).all(1)
        logp[empty] = -INF
        p = logp.exp()
        h = -torch.nan_to_num(p * logp, nan=0.0).sum(1)
        a = state["taken"][rows].long()
        lp = logp[torch.arange(len(a), device="cuda"), a.clamp(0, v - 1)]
        lp[(a < 0) | (a >= v)] = 0.0
        out["logprob"][rows], out["entropy"][rows] = lp, h
        if top:
            out["top_logprobs"][rows] = logp.topk(top, dim=1).values
        if case["kind"] == "learn":
            gl, gh = state["grad_logprob"][rows].double(), state["grad_entropy"][rows].double()
            gl = gl * ((a >= 0) & (a < v))
            one = torch.zeros_like(p)
            one[torch.arange(len(a), device="cuda"), a.clamp(0, v - 1)] = 1.0
            to_h = torch.nan_to_num(-p * (logp + h[:, None]), nan=0.0)
            grad = (gl[:, None] * (one - p) + gh[:, None] * to_h) / case["temperature"]
            grad[empty] = 0.0
            if "legal" in state:
                grad[state["legal"][rows] == 0] = 0.0
            out["grad"][rows] = grad
    return out


def _exact_adamw(state):
    """The codes' exact values are what they are rounded from."""
    case, t = state["case"], state["t"] + 1
    g = state["grad"].double()
    if case["clip"]:
        g *= min(1.0, 1.0 / (float(torch.linalg.vector_norm(g)) + 1e-6))
    m, v = state["m"].double(), state["v"].double()
    if case["bits"] == 8:
        m *= state["m_scale"].double().repeat_interleave(BLOCK)
        v = (v * state["v_scale"].double().repeat_interleave(BLOCK)) ** 2
    m = m * BETA1 + g * (1 - BETA1)
    v = v * BETA2 + g ** 2 * (1 - BETA2)
    del g
    p = state["master" if case["master"] else "param"].double()
    decay = state["decays"].double()[state["of_block"]].repeat_interleave(BLOCK)
    p = p - LR * decay * p - LR * m / (1 - BETA1 ** t) / ((v / (1 - BETA2 ** t)) ** 0.5 + EPS)
    out = dict(param=p)
    if case["master"]:
        out["master"] = p
    if case["bits"] == 32:
        return dict(out, m=m, v=v)
    for key, x in (("m", m), ("v", v ** 0.5)):
        scale = x.view(-1, BLOCK).abs().max(1).values / E4M3_MAX
        out[key + "_scale"] = scale
        out[key] = x / torch.where(scale > 0, scale, 1.0).repeat_interleave(BLOCK)
    return out
