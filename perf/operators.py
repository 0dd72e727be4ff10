"""Cases and plain forms of the model operators (include/hccl_model_ops.h, hccl_amd/model_ops.py).

Four operators that stand between a model and the collectives:

  log_probs       log probabilities of given tokens, entropy and the most likely alternatives of every row of logits
                  whose vocabulary is split across the ranks; every rank receives the results
  log_probs_grad  its gradient with respect to one rank's part of the logits
  grad_norm       2-norm over all gradient tensors of all ranks, and the factor that clips it
  adamw           one AdamW step over many tensors, with states in 32 bits or in FP8 blocks of 256

`own` chooses between the plain form (elementary torch operations, 32 bits, 64 for long sums) and the calls a user
makes of the framework.  Those go to a stream of their own, as the library takes no null stream, and are ordered by the
device alone: whoever calls `prepare` and `run` on another stream synchronizes the device between the two, before the
results are read, and before a state is dropped.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BLOCK = 256            # elements that share a scale of an 8-bit state
FP8_MAX = 448.0        # largest value of float8_e4m3fn
FP8_MIN = 2.0 ** -9    # smallest positive one
BETA1, BETA2, EPS, DECAY = 0.9, 0.95, 1e-8, 0.1
IGNORED = -100


def listed():
    return [
        # one sequence that is being decoded on one GPU: the smallest call, latency counts
        {"name": "log_probs one token", "op": "log_probs", "ranks": 1, "tokens": 1, "vocab": 32768, "dtype": "bf16",
         "top": 5, "padded": True, "masked": False, "scale": 1.0},
        # a serving batch that is being decoded, its vocabulary split over eight ranks, the usual twenty alternatives
        {"name": "log_probs decode, 8 ranks", "op": "log_probs", "ranks": 8, "tokens": 64, "vocab": 131072,
         "dtype": "bf16", "top": 20, "padded": True, "masked": True, "scale": 1.25},
        # scoring whole sequences for a policy gradient, a long batch of prompts and answers
        {"name": "log_probs 4096 tokens", "op": "log_probs", "ranks": 1, "tokens": 4096, "vocab": 131072,
         "dtype": "bf16", "top": 0, "padded": True, "masked": False, "scale": 1.0},
        # evaluation with alternatives: odd vocabulary, uneven parts, rows that begin on any element
        {"name": "log_probs ragged fp32", "op": "log_probs", "ranks": 3, "tokens": 777, "vocab": 50001,
         "dtype": "fp32", "top": 8, "padded": False, "masked": True, "scale": 0.5},
        # a small micro-batch's loss over two ranks
        {"name": "log_probs_grad 16 tokens", "op": "log_probs_grad", "ranks": 2, "tokens": 16, "vocab": 32768,
         "dtype": "fp16", "top": 0, "padded": True, "masked": False, "scale": 1.0},
        # the loss of a training step, its vocabulary split over eight ranks
        {"name": "log_probs_grad 4096 tokens", "op": "log_probs_grad", "ranks": 8, "tokens": 4096, "vocab": 131072,
         "dtype": "bf16", "top": 0, "padded": True, "masked": True, "scale": 1.0},
        # distillation from the alternatives: a gradient into the top values too, odd sizes throughout
        {"name": "log_probs_grad ragged", "op": "log_probs_grad", "ranks": 3, "tokens": 1001, "vocab": 50001,
         "dtype": "bf16", "top": 8, "padded": False, "masked": False, "scale": 0.5},
        # the gradients of a small model (biases, norms, a few matrices) on two ranks
        {"name": "grad_norm small", "op": "grad_norm", "ranks": 2, "tensors": 12, "elements": 40000, "dtype": "fp32"},
        # eight ranks that hold an eighth each of the gradients of half a billion parameters
        {"name": "grad_norm 8 ranks", "op": "grad_norm", "ranks": 8, "tensors": 120, "elements": 1 << 26,
         "dtype": "bf16"},
        # a small model or an adapter, all in 32 bits
        {"name": "adamw small fp32", "op": "adamw", "tensors": 24, "elements": 300000, "param": "fp32", "grad": "fp32",
         "master": False, "state": "fp32", "step": 1},
        # one rank's shard in mixed precision: 32-bit master weights and states, 16-bit weights and gradients
        {"name": "adamw shard mixed", "op": "adamw", "tensors": 300, "elements": 1 << 27, "param": "bf16",
         "grad": "bf16", "master": True, "state": "fp32", "step": 1000},
        # the same shard with states in 8 bits
        {"name": "adamw shard fp8 states", "op": "adamw", "tensors": 300, "elements": 1 << 27, "param": "bf16",
         "grad": "bf16", "master": True, "state": "fp8", "step": 1000},
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["log_probs", "log_probs_grad", "grad_norm", "adamw"])
    if op in ("log_probs", "log_probs_grad"):
        vocab = _log_uniform(rng, 1000, 160000)
        top = rng.choice([0, 0, 1, 5, 8, 20, 32])
        most = (1 << 26 if top else 1 << 28) // vocab
        return {"op": op, "ranks": rng.choice([1, 2, 3, 4, 8]), "tokens": _log_uniform(rng, 1, min(4096, most)),
                "vocab": vocab, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "top": top,
                "padded": rng.random() < 0.5, "masked": rng.random() < 0.3, "scale": rng.choice([1.0, 0.5, 1.25])}
    if op == "grad_norm":
        ranks = rng.choice([1, 2, 3, 4, 8])
        return {"op": op, "ranks": ranks, "tensors": _log_uniform(rng, 1, 300),
                "elements": _log_uniform(rng, 1000, (1 << 28) // ranks), "dtype": rng.choice(["bf16", "fp16", "fp32"])}
    param = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    return {"op": op, "tensors": _log_uniform(rng, 1, 400), "elements": _log_uniform(rng, 1000, 1 << 26),
            "param": param, "grad": rng.choice([param, "fp32"]), "master": param != "fp32" and rng.random() < 0.6,
            "state": rng.choice(["fp32", "fp8"]), "step": rng.choice([1, 2, 17, 1000, 100000])}


def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    if case["op"] == "log_probs":
        n = case["tokens"] * case["vocab"]
        out = case["tokens"] * (12 + 12 * case["top"])
        return {"bytes": n * size[case["dtype"]] + case["tokens"] * 8 + case["ranks"] * out, "flops": 8 * n}
    if case["op"] == "log_probs_grad":
        n = case["tokens"] * case["vocab"]
        return {"bytes": 2 * n * size[case["dtype"]] + case["tokens"] * (24 + 12 * case["top"]), "flops": 8 * n}
    if case["op"] == "grad_norm":
        n = case["ranks"] * case["elements"]
        return {"bytes": n * size[case["dtype"]] + 8 * case["ranks"], "flops": 2 * n}
    state = 8 if case["state"] == "fp32" else 2 + 8 / BLOCK
    each = size[case["grad"]] + 2 * state + (8 + size[case["param"]] if case["master"] else 2 * size[case["param"]])
    return {"bytes": each * case["elements"], "flops": 16 * case["elements"]}


# ---- inputs ---------------------------------------------------------------------------------------------------
def _parts(case):
    """(first index, count) of every rank's part of the vocabulary: equal parts, the last one shorter."""
    each = -(-case["vocab"] // case["ranks"])
    starts = [min(case["vocab"], r * each) for r in range(case["ranks"] + 1)]
    return [(a, b - a) for a, b in zip(starts, starts[1:])]


def _tensor_sizes(case):
    """Element counts of the case's tensors: vectors, matrices and a few large tables, odd counts among them."""
    rng = random.Random(7 * case["tensors"] + case["elements"])
    weights = [rng.choice([1, 40, 40, 300, 300, 2500]) * rng.uniform(0.5, 1.0) for _ in range(case["tensors"])]
    left, sizes = case["elements"], []
    for i, w in enumerate(weights):
        n = int(left * w / sum(weights[i:])) if i + 1 < len(weights) else left
        sizes.append(n)
        left -= n
    return sizes


def _layout(case):
    """(offset, count) of every tensor in one buffer, and the buffer's length: tensors begin on whole blocks."""
    at, out = 0, []
    for n in _tensor_sizes(case):
        out.append((at, n))
        at += -(-n // BLOCK) * BLOCK
    return out, max(at, BLOCK)


def _fill(layout, length, make):
    """A buffer with `make(length)` in the tensors and zeros in the gaps between them."""
    inside = torch.zeros(length + 1, dtype=torch.int32, device="cuda")
    edges = torch.tensor(layout, dtype=torch.int64, device="cuda")
    one = torch.ones(len(layout), dtype=torch.int32, device="cuda")
    inside.index_add_(0, edges[:, 0], one)
    inside.index_add_(0, edges[:, 0] + edges[:, 1], -one)
    inside = inside.cumsum(0)[:length] > 0
    x = make(length)
    return x.masked_fill_(~inside, 0)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype)

    if case["op"] in ("log_probs", "log_probs_grad"):
        return _prepare_logits(case, gen, normal)
    layout, length = _layout(case)
    if case["op"] == "grad_norm":
        dtype = DTYPES[case["dtype"]]
        grads = torch.stack([_fill(layout, length, lambda n: normal(n, dtype=dtype).mul_(1e-2))
                             for _ in range(case["ranks"])])
        return {"case": case, "layout": layout, "grads": grads,
                "result": torch.zeros(case["ranks"], 2, device="cuda"), "max_norm": 1.0, "scale": 0.25}
    weights = _fill(layout, length, lambda n: normal(n).mul_(0.02))
    # gradients of an embedding are zero in most rows: a tenth of the blocks has none
    quiet = (torch.rand(length // BLOCK, generator=gen, device="cuda") < 0.1).repeat_interleave(BLOCK)
    grads = _fill(layout, length, lambda n: normal(n).mul_(1e-3)).masked_fill_(quiet, 0)
    state = {"case": case, "layout": layout, "lr": 3e-4,
             "param": weights.to(DTYPES[case["param"]]), "grad": grads.to(DTYPES[case["grad"]]),
             "clip": torch.tensor([2.0, 0.5], device="cuda")}
    if case["master"]:
        state["master"] = weights
    if case["step"] == 1:
        m = torch.zeros(length, device="cuda")
        v = torch.zeros(length, device="cuda")
    else:
        m = _fill(layout, length, lambda n: normal(n).mul_(2e-4))
        v = (m * 2 + 1e-6 * (m != 0)).square()
    if case["state"] == "fp32":
        return dict(state, m=m, v=v)
    m, m_scale = _to_fp8(m)
    v, v_scale = _root_to_fp8(v)
    return dict(state, m=m, v=v, m_scale=m_scale, v_scale=v_scale)


def _prepare_logits(case, gen, normal):
    tokens, dtype = case["tokens"], DTYPES[case["dtype"]]
    parts = _parts(case)
    likely = torch.randint(0, case["vocab"], (tokens,), generator=gen, device="cuda")
    other = torch.randint(0, case["vocab"], (tokens,), generator=gen, device="cuda")
    chance = torch.rand(tokens, generator=gen, device="cuda")
    given = torch.where(chance < 0.7, likely, other)
    if tokens >= 16:
        given = given.masked_fill(chance > 0.95, IGNORED)     # padding and prompts that carry no loss
    boost = 6.0 + 8.0 * torch.rand(tokens, generator=gen, device="cuda")
    logits = []
    for start, count in parts:
        stride = -(-count // 64) * 64 if case["padded"] else count
        x = normal(tokens, max(stride, 1), dtype=dtype).mul_(2.0)
        here = (likely >= start) & (likely < start + count)
        rows = here.nonzero().squeeze(1)
        x[rows, likely[rows] - start] = boost[rows].to(dtype)
        if case["masked"]:
            keep = case["vocab"] - case["vocab"] // 100        # the padding of the vocabulary can not be chosen
            x[:, max(0, min(count, keep - start)):count] = -math.inf
            if tokens > 1:                                    # a grammar that leaves one choice
                x[1] = -math.inf
                if start <= 17 < start + count:
                    x[1, 17 - start] = 1.0
        logits.append(x)
    if case["masked"]:
        given = torch.where(given < case["vocab"] - case["vocab"] // 100, given, given - case["vocab"] // 100)
        if tokens > 1:
            given[1] = 17
    ranks, top = case["ranks"], case["top"]
    state = {"case": case, "parts": parts, "logits": logits, "tokens": given}
    if case["op"] == "log_probs":
        def empty(*shape, dtype=torch.float32):
            return torch.zeros(ranks, *shape, device="cuda", dtype=dtype)
        state["out"] = {"log_probs": empty(tokens), "lse": empty(tokens), "entropy": empty(tokens)}
        if top:
            state["out"].update(top_values=empty(tokens, top), top_ids=empty(tokens, top, dtype=torch.int64))
        return state
    forward = _log_probs(case, parts, logits, given)          # what the forward pass left behind
    state["lse"], state["entropy"] = forward["lse"], forward["entropy"]
    state["grad_log_probs"] = normal(tokens).div_(tokens).masked_fill_(given < 0, 0)
    state["grad_entropy"] = normal(tokens).mul_(0.01 / tokens).masked_fill_(given < 0, 0)
    if top:
        state["top_ids"] = forward["top_ids"].contiguous()
        state["grad_top"] = normal(tokens, top).mul_(0.1 / tokens)
    state["grads"] = [torch.zeros_like(x) for x in logits]
    return state


# ---- plain forms ----------------------------------------------------------------------------------------------
def _whole(parts, logits):
    return torch.cat([x[:, :count] for (_, count), x in zip(parts, logits)], 1)


def _log_probs(case, parts, logits, given):
    """One row of results per token (not per rank)."""
    raw = _whole(parts, logits).float()
    x = raw * case["scale"]
    y = x - x.amax(1, keepdim=True)
    e = y.exp()
    total = e.sum(1)
    log_total = total.log()
    weighted = torch.where(e > 0, e * y, 0.0).sum(1)
    token = y.gather(1, given.clamp(min=0)[:, None])[:, 0] - log_total
    out = {"log_probs": torch.where(given >= 0, token, 0.0), "lse": x.amax(1) + log_total,
           "entropy": log_total - weighted / total}
    if case["top"]:
        bits = (raw + 0.0).view(torch.int32)                   # + 0.0: the two zeros are one value
        order = torch.where(bits >= 0, bits, bits ^ 0x7FFFFFFF).long() << 32
        order += 0x7FFFFFFF - torch.arange(case["vocab"], device="cuda")   # of equal logits the first
        best = order.topk(case["top"], 1).values
        out["top_ids"] = 0x7FFFFFFF - (best & 0x7FFFFFFF)
        out["top_values"] = y.gather(1, out["top_ids"]) - log_total[:, None]
    return out


def _plain_log_probs(state):
    got = _log_probs(state["case"], state["parts"], state["logits"], state["tokens"])
    return {k: v.expand(state["case"]["ranks"], *v.shape) for k, v in got.items()}


def _plain_log_probs_grad(state):
    case, given = state["case"], state["tokens"]
    log_p = _whole(state["parts"], state["logits"]).float() * case["scale"] - state["lse"][:, None]
    p = log_p.exp()
    valid = (given >= 0).float() * state["grad_log_probs"]
    into = valid + (state["grad_top"].sum(1) if case["top"] else 0)
    d = -p * (into[:, None] + state["grad_entropy"][:, None] * (log_p.clamp(min=-1000) + state["entropy"][:, None]))
    d.scatter_add_(1, given.clamp(min=0)[:, None], valid[:, None])
    if case["top"]:
        d.scatter_add_(1, state["top_ids"], state["grad_top"])
    d = (d * case["scale"]).to(DTYPES[case["dtype"]])
    return [d[:, start:start + count] for start, count in state["parts"]]


def _plain_grad_norm(state):
    norm = abs(state["scale"]) * state["grads"].double().square().sum().sqrt()
    factor = state["scale"] * (state["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    return torch.stack([norm, factor]).float().expand(state["case"]["ranks"], 2)


def _to_fp8(m):
    m = m.view(-1, BLOCK)
    most = m.abs().amax(1, keepdim=True)
    code = torch.where(most > 0, m * (FP8_MAX / most), 0.0)
    return code.to(torch.float8_e4m3fn).view(-1), (most / FP8_MAX).view(-1)


def _root_to_fp8(v):
    """The square root is what is stored (half the range), and a value above zero stays above zero."""
    root = v.sqrt().view(-1, BLOCK)
    most = root.amax(1, keepdim=True)
    code = torch.where(root > 0, (root * (FP8_MAX / most)).clamp(min=FP8_MIN), 0.0)
    return code.to(torch.float8_e4m3fn).view(-1), (most / FP8_MAX).view(-1)


def _plain_adamw(state):
    case, step, lr = state["case"], state["case"]["step"], state["lr"]
    fp8 = case["state"] == "fp8"
    weights = state["master"] if case["master"] else state["param"].float()
    g = state["grad"].float() * state["clip"][1]
    m, v = state["m"], state["v"]
    if fp8:
        m = (m.float().view(-1, BLOCK) * state["m_scale"][:, None]).view(-1)
        v = (v.float().view(-1, BLOCK) * state["v_scale"][:, None]).view(-1).square()
    m = m * BETA1 + g * (1 - BETA1)
    v = v * BETA2 + g * g * (1 - BETA2)
    denominator = v.sqrt() / math.sqrt(1 - BETA2 ** step) + EPS
    weights = weights * (1 - lr * DECAY) - m / denominator * (lr / (1 - BETA1 ** step))
    state["param"].copy_(weights)
    if case["master"]:
        state["master"].copy_(weights)
    if fp8:
        m, m_scale = _to_fp8(m)
        v, v_scale = _root_to_fp8(v)
        state["m_scale"].copy_(m_scale)
        state["v_scale"].copy_(v_scale)
    state["m"].copy_(m)
    state["v"].copy_(v)
    return _updated(state)


def _updated(state):
    return {k: state[k] for k in ("param", "master", "m", "v", "m_scale", "v_scale") if k in state}


# ---- the framework's calls --------------------------------------------------------------------------------------
_worlds = {}


def _world(ranks):
    """The communicators of a world of that many ranks and the stream its calls go to, as a program keeps them.  (A program
    that runs on that stream throughout needs no other order; events to and from the null stream take 35 us a pass.)"""
    import hccl_amd
    if ranks not in _worlds:
        _worlds[ranks] = (hccl_amd.comm_init_all(ranks), _worlds[min(_worlds)][1] if _worlds else torch.cuda.Stream())
    return _worlds[ranks]


def _code(name):
    from hccl_amd import HcclDataType
    return {"bf16": HcclDataType.BFP16, "fp16": HcclDataType.FP16, "fp32": HcclDataType.FP32,
            "fp8": HcclDataType.FP8E4M3}[name]


def _own_log_probs(state):
    import hccl_amd
    from hccl_amd import model_ops
    case, out = state["case"], state["out"]
    comms, stream = _world(case["ranks"])
    top = case["top"]
    if "workspace" not in state:      # a program keeps it for all calls of this size
        size = model_ops.token_log_probs_workspace(case["tokens"], case["vocab"], top)
        state["workspace"] = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda") if size else None
    space = state["workspace"]
    with hccl_amd.group():
        for r, (start, count) in enumerate(state["parts"]):
            x = state["logits"][r]
            model_ops.token_log_probs(
                comms[r], x, case["tokens"], start, count, state["tokens"], out["log_probs"][r],
                data_type=_code(case["dtype"]), row_stride=x.stride(0), scale=case["scale"], lse=out["lse"][r],
                entropy=out["entropy"][r], top_count=top, top_values=out["top_values"][r] if top else None,
                top_ids=out["top_ids"][r] if top else None, workspace=space,
                workspace_bytes=space.numel() if space is not None else 0, stream=stream)
    return out


def _own_log_probs_grad(state):
    from hccl_amd import model_ops
    case, top = state["case"], state["case"]["top"]
    comms, stream = _world(case["ranks"])
    for r, (start, count) in enumerate(state["parts"]):
        x, d = state["logits"][r], state["grads"][r]
        model_ops.token_log_probs_grad(
            comms[r], x, case["tokens"], start, count, state["tokens"], state["lse"], state["grad_log_probs"], d,
            data_type=_code(case["dtype"]), row_stride=x.stride(0), grad_row_stride=d.stride(0), scale=case["scale"],
            entropy=state["entropy"], grad_entropy=state["grad_entropy"], top_count=top,
            top_ids=state["top_ids"] if top else None, grad_top_values=state["grad_top"] if top else None,
            stream=stream)
    return [d[:, :count] for (_, count), d in zip(state["parts"], state["grads"])]


def _own_grad_norm(state):
    import hccl_amd
    from hccl_amd import model_ops
    case = state["case"]
    comms, stream = _world(case["ranks"])
    if "tensors" not in state:        # a program describes its gradient buffers once
        state["tensors"] = [model_ops.norm_tensors([(row[at:at + n], n, _code(case["dtype"]))
                                                    for at, n in state["layout"]]) for row in state["grads"]]
        size = model_ops.grad_norm_workspace(case["ranks"] * case["tensors"])
        state["workspace"] = torch.empty(size, dtype=torch.uint8, device="cuda")
    with hccl_amd.group():
        for r in range(case["ranks"]):
            model_ops.grad_norm(comms[r], state["tensors"][r], state["max_norm"], state["result"][r],
                                scale=state["scale"], workspace=state["workspace"],
                                workspace_bytes=state["workspace"].numel(), stream=stream)
    return state["result"]


def _own_adamw(state):
    from hccl_amd import model_ops
    case = state["case"]
    comms, stream = _world(1)
    if "tensors" not in state:        # a program describes its tensors once
        fp8 = case["state"] == "fp8"
        state["tensors"] = model_ops.adamw_tensors([
            dict(param=state["param"][at:], grad=state["grad"][at:], exp_avg=state["m"][at:], exp_avg_sq=state["v"][at:],
                 count=n, param_type=_code(case["param"]), grad_type=_code(case["grad"]),
                 master=state["master"][at:] if case["master"] else None,
                 exp_avg_scale=state["m_scale"][at // BLOCK:] if fp8 else None,
                 exp_avg_sq_scale=state["v_scale"][at // BLOCK:] if fp8 else None) for at, n in state["layout"]])
    model_ops.adamw(comms[0], state["tensors"], step=case["step"], lr=state["lr"], beta1=BETA1, beta2=BETA2, eps=EPS,
                    weight_decay=DECAY, state_type=_code(case["state"]), clip=state["clip"], stream=stream)
    return _updated(state)


def run(state):
    op = state["case"]["op"]
    if own:
        return {"log_probs": _own_log_probs, "log_probs_grad": _own_log_probs_grad, "grad_norm": _own_grad_norm,
                "adamw": _own_adamw}[op](state)
    return {"log_probs": _plain_log_probs, "log_probs_grad": _plain_log_probs_grad, "grad_norm": _plain_grad_norm,
            "adamw": _plain_adamw}[op](state)


# ---- 64 bits ----------------------------------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "log_probs":
        raw = torch.cat([x[:, :n].double() for (_, n), x in zip(state["parts"], state["logits"])], 1)
        log_p = torch.log_softmax(raw * case["scale"], 1)
        rows = torch.arange(case["tokens"], device="cuda")
        given = state["tokens"]
        out = {"log_probs": torch.where(given >= 0, log_p[rows, given.clamp(min=0)], 0.0),
               "lse": torch.logsumexp(raw * case["scale"], 1),
               "entropy": torch.special.entr(log_p.exp()).sum(1)}
        if case["top"]:
            ids = torch.sort(raw + 0.0, dim=1, descending=True, stable=True).indices[:, :case["top"]]
            out.update(top_ids=ids, top_values=log_p.gather(1, ids))
        return {k: v.expand(case["ranks"], *v.shape) for k, v in out.items()}
    if case["op"] == "log_probs_grad":
        raw = [x[:, :n].double().requires_grad_() for (_, n), x in zip(state["parts"], state["logits"])]
        log_p = torch.log_softmax(torch.cat(raw, 1) * case["scale"], 1)
        given = state["tokens"]
        finite = torch.where(log_p > -1000, log_p, 0.0)
        entropy = -(finite * log_p.exp()).sum(1)
        token = log_p.gather(1, given.clamp(min=0)[:, None])[:, 0]
        loss = (torch.where(given >= 0, token, 0.0) * state["grad_log_probs"].double()).sum()
        loss = loss + (entropy * state["grad_entropy"].double()).sum()
        if case["top"]:
            loss = loss + (log_p.gather(1, state["top_ids"]) * state["grad_top"].double()).sum()
        return list(torch.autograd.grad(loss, raw))
    if case["op"] == "grad_norm":
        norm = 0.25 * torch.linalg.vector_norm(state["grads"].double())
        factor = 0.25 * torch.minimum(torch.ones_like(norm), 1.0 / (norm + 1e-6))
        return torch.stack([norm, factor]).expand(case["ranks"], 2)
    return _exact_adamw(case, state)


def _exact_adamw(case, state):
    t = case["step"]
    w = (state["master"] if case["master"] else state["param"]).double()
    g = state["grad"].double() / 2
    m, v = state["m"].double(), state["v"].double()
    if case["state"] == "fp8":
        m = m * state["m_scale"].double().repeat_interleave(BLOCK)
        v = (v * state["v_scale"].double().repeat_interleave(BLOCK)) ** 2
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * g ** 2
    unbiased_m, unbiased_v = m / (1 - BETA1 ** t), v / (1 - BETA2 ** t)
    w = w - state["lr"] * DECAY * w - state["lr"] * unbiased_m / (unbiased_v ** 0.5 + EPS)
    out = {"param": w, "m": m, "v": v}
    if case["master"]:
        out["master"] = w
    if case["state"] == "fp8":
        root = v.sqrt()
        for name, x in (("m", m), ("v", root)):
            most = x.abs().view(-1, BLOCK).amax(1)
            out[name + "_scale"] = most / FP8_MAX
            unit = FP8_MAX / torch.where(most > 0, most, 1.0).repeat_interleave(BLOCK)
            out[name] = x * unit
        out["v"] = torch.where(root > 0, out["v"].clamp(min=FP8_MIN), 0.0)
    return out
