"""GPU tests of the model operators (include/hccl_model_ops.h) against plain 64-bit implementations.

Tolerances are derived from the arithmetic, not fitted.  U = 2^-24 is half a step of a 32-bit float; a rounding to a type
with step eps is off by at most eps / 2 of the value.  Sums of n positive 32-bit terms are off by at most n U relative; a
lane of the log-probability kernel adds at most ceil(V / 2048) * 8 + 64 terms (256 lanes, vectors of eight, partial vectors
per part), then log2(256) + 64 partial sums are joined."""
import math

import numpy as np
import pytest

import hccl_amd
from hccl_amd import HcclDataType as DT
from hccl_amd import HcclReduceOp as OP
from hccl_amd import model_ops

from gpu_util import World, require_library_on_gpu

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TORCH = {DT.FP32: torch.float32, DT.BFP16: torch.bfloat16, DT.FP16: torch.float16, DT.INT32: torch.int32,
         DT.INT64: torch.int64}
FILL = 77.0


@pytest.fixture(scope="module", autouse=True)
def _native_library():
    require_library_on_gpu()
    model_ops.lib()


@pytest.fixture(scope="module")
def worlds():
    made = {}

    def get(n):
        if n not in made:
            made[n] = World(n)
        return made[n]
    yield get
    for w in made.values():
        w.close()


def rng_tensor(seed, *shape, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g) * scale


def split(vocab, ranks, seed=0):
    """Uneven parts of a vocabulary, an empty one among them where there are three ranks or more."""
    cuts = sorted(np.random.default_rng(seed).integers(0, vocab + 1, ranks - 1).tolist())
    if ranks >= 3:
        cuts[1] = cuts[0]
    edges = [0] + sorted(cuts) + [vocab]
    return [(a, b - a) for a, b in zip(edges, edges[1:])]


class Rows:
    """Logits [T, V] of a type, dealt to ranks as parts that start on any element and whose rows are any distance apart,
    and the outputs of every rank.  With `tight` a part's memory ends with its last element."""

    def __init__(self, x, dtype, ranks, top=0, token_type=DT.INT64, parts=None, pad=3, offset=1, tight=False):
        self.t, self.v = x.shape
        self.dtype, self.top, self.token_type = dtype, top, token_type
        self.x = x.to(TORCH[dtype])
        self.parts = parts or split(self.v, ranks, self.t + self.v)
        self.shards = []
        for start, count in self.parts:
            stride = count + pad
            room, whole = self.room(offset, stride, count if tight else stride)
            whole[:, :count] = self.x[:, start:start + count].cuda()
            self.shards.append(whole)
        n = len(self.parts)
        self.log_probs = [torch.full((self.t + 1,), FILL, device="cuda") for _ in range(n)]
        self.lse = [torch.full((self.t + 1,), FILL, device="cuda") for _ in range(n)]
        self.entropy = [torch.full((self.t + 1,), FILL, device="cuda") for _ in range(n)]
        self.values = [torch.full((self.t * top + 1,), FILL, device="cuda") for _ in range(n)]
        self.ids = [torch.full((self.t * top + 1,), 77, device="cuda", dtype=TORCH[token_type]) for _ in range(n)]

    def room(self, offset, stride, width):
        """Memory of T rows `stride` apart, of which `width` elements are looked at, that ends with the last of these."""
        room = torch.full((offset + (self.t - 1) * stride + width,), FILL, dtype=TORCH[self.dtype], device="cuda")
        return room, room.as_strided((self.t, width), (stride, 1), offset)

    def run(self, w, tokens, scale=1.0, streams=None, space=None):
        tokens = tokens.to(TORCH[self.token_type]).cuda()
        size = model_ops.token_log_probs_workspace(self.t, self.v, self.top)
        space = torch.full((max(size, 1),), 255, dtype=torch.uint8, device="cuda") if space is None else space
        torch.cuda.synchronize()
        with hccl_amd.group():
            for r, (start, count) in enumerate(self.parts):
                s = self.shards[r]
                model_ops.token_log_probs(
                    w.comms[r], s if count else None, self.t, start, count, tokens, self.log_probs[r],
                    data_type=self.dtype, token_type=self.token_type, row_stride=s.stride(0), scale=scale, lse=self.lse[r],
                    entropy=self.entropy[r], top_count=self.top, top_values=self.values[r], top_ids=self.ids[r],
                    workspace=space, workspace_bytes=size, stream=w.stream if streams is None else streams[r])
        torch.cuda.synchronize()
        for r in range(len(self.parts)):       # every rank has the same results, and nothing behind them
            for got in (self.log_probs, self.lse, self.entropy, self.values, self.ids):
                assert torch.equal(got[r].nan_to_num(9e9), got[0].nan_to_num(9e9)), r
                assert float(got[r][-1]) == 77
        k = self.top
        return (self.log_probs[0][:-1].cpu().double(), self.lse[0][:-1].cpu().double(), self.entropy[0][:-1].cpu().double(),
                self.values[0][:-1].view(self.t, k).cpu().double() if k else None,
                self.ids[0][:-1].view(self.t, k).cpu().long() if k else None)


def reference(x, tokens, scale, top):
    """The definition, in 64 bits on the CPU."""
    raw = x.double()
    z = raw * float(np.float32(scale))
    most = z.amax(1, keepdim=True)
    shift = torch.where(most > -math.inf, most, 0.0)
    e = (z - shift).exp()
    s = e.sum(1)
    lse = shift[:, 0] + s.log()
    log_p = torch.where(s[:, None] > 0, (z - shift) - s.log()[:, None], -math.inf)
    p = log_p.exp()
    entropy = -torch.where(p > 0, p * log_p, 0.0).sum(1)
    lp = torch.where(tokens >= 0, log_p.gather(1, tokens.clamp(0, x.shape[1] - 1)[:, None])[:, 0], 0.0)
    lp = torch.where(tokens >= x.shape[1], math.nan, lp)
    ids = torch.sort(raw + 0.0, dim=1, descending=True, stable=True).indices[:, :top]
    return lp, lse, entropy, log_p.gather(1, ids), ids, log_p


def terms(v):
    """Additions on the way of one term of a row's sums, see above, and twenty roundings that do not grow with V."""
    return math.ceil(v / 2048) * 8 + 64 + 8 + 64 + 20


def check_rows(rows, got, tokens, scale):
    lp, lse, entropy, values, ids, _ = reference(rows.x, tokens, scale, rows.top)
    n = terms(rows.v)
    size = lambda a: torch.where(a.isfinite(), a.abs(), 0.0)  # noqa: E731
    # log p = scale (x - m) - ln s: s is off by n U relative plus the exponent's error: y = (x - m) c is rounded twice and c
    # once, |y| 3 U, times e^-|y| at most 3 U; one exponential, 2 U; the rest are roundings of the terms themselves.
    sums = (n + 8) * U
    # the entropy's second term t / s: the same sums, of terms y e^y below 0.54 each in magnitude, relative to s
    for name, a, b, tol in (("log_probs", got[0], lp, sums + 4 * U * (size(lp) + size(lse))),
                            ("lse", got[1], lse, sums + 4 * U * size(lse)),
                            ("entropy", got[2], entropy, 3 * sums * (1 + size(entropy)) + 4 * U * math.log(rows.v + 1))):
        same = (a == b) | (a.isnan() & b.isnan())
        assert bool((same | ((a - b).abs() <= tol)).all()), (name, float((a - b).abs().nan_to_num(0).max()))
    if rows.top:
        assert torch.equal(got[4], ids)
        tol = sums + 4 * U * (size(values) + size(lse)[:, None])
        same = (got[3] == values) | (got[3].isnan() & values.isnan())
        assert bool((same | ((got[3] - values).abs() <= tol)).all())


def given(t, v, seed):
    tokens = torch.randint(0, v, (t,), generator=torch.Generator().manual_seed(seed))
    if t > 2:
        tokens[1], tokens[2] = -100, -1
    if t > 5:
        tokens[3], tokens[4], tokens[5] = 0, v - 1, v      # the last is none of the vocabulary
    return tokens


# ---- log probabilities ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [DT.FP32, DT.BFP16, DT.FP16])
@pytest.mark.parametrize("t,v,ranks,top", [
    (1, 1, 1, 1), (1, 7, 1, 7), (2, 9, 2, 3), (3, 33, 2, 32), (7, 255, 3, 5), (5, 2049, 1, 32), (6, 4099, 3, 20),
    (130, 1000, 4, 1), (2, 8192, 1, 8), (1, 40001, 2, 32), (3, 131072, 8, 20), (1, 70000, 1, 0), (64, 20011, 3, 9),
    (1025, 77, 2, 3), (1, 300000, 1, 5)])
def test_log_probs(worlds, dtype, t, v, ranks, top):
    x = rng_tensor(t * 7 + v, t, v, scale=3.0)
    x[:, v // 3] += 9.0                                    # a likely entry
    tokens = given(t, v, 5)
    scale = (1.0, 0.7, 1.3)[(t + v) % 3]
    rows = Rows(x, dtype, ranks, top, DT.INT32 if v % 2 else DT.INT64)
    check_rows(rows, rows.run(worlds(ranks), tokens, scale), tokens, scale)


@pytest.mark.parametrize("parts", [[(0, 0), (0, 5), (5, 0), (5, 4096)], [(0, 8), (8, 8), (16, 8), (24, 2)],
                                   [(i * 40, 40) for i in range(64)], [(0, 9000)] + [(9000, 0)] * 7])
def test_parts_of_any_size(worlds, parts):
    v = sum(c for _, c in parts)
    x = rng_tensor(len(parts), 9, v, scale=2.0)
    tokens = given(9, v, 3)
    rows = Rows(x, DT.BFP16, len(parts), 12, parts=parts)
    check_rows(rows, rows.run(worlds(len(parts)), tokens), tokens, 1.0)


@pytest.mark.parametrize("dtype", [DT.FP32, DT.BFP16, DT.FP16])
@pytest.mark.parametrize("t,v", [(12, 5000), (1100, 300), (12, 70000)])
def test_masked_rows(worlds, dtype, t, v):
    """Masks of -inf and of the type's lowest value, up to rows that nothing is left of; both zeros; NaN and +inf."""
    x = rng_tensor(v, t, v, scale=2.0)
    low = torch.finfo(TORCH[dtype]).min
    x[0] = -math.inf                                       # nothing left
    x[1] = low                                             # all equal: uniform
    x[2] = -math.inf
    x[2, v - 3] = -5.0                                     # one entry left
    x[3, ::2] = -math.inf
    x[4, : v - 2] = low
    x[5] = low
    x[5, 3:9] = -math.inf
    x[6] = 0.0                                             # ties throughout, both zeros
    x[6, ::3] = -0.0
    x[7, v // 2] = math.nan
    x[8, 17] = math.inf
    x[9, 5] = torch.finfo(TORCH[dtype]).max
    x[10] = -math.inf
    x[10, v - 1] = low
    x[11, :] = math.nan
    tokens = torch.full((t,), 2)
    tokens[2], tokens[7] = v - 3, -100
    rows = Rows(x, dtype, 2, 16)
    got = rows.run(worlds(2), tokens, 1.0)
    good = [i for i in range(t) if i not in (7, 8, 11)]
    part = Rows(x[good], dtype, 2, 16)
    check_rows(part, tuple(g[good] for g in got), tokens[good], 1.0)
    for i in (7, 8, 11):
        assert got[1][i].isnan() and got[2][i].isnan() and bool(got[3][i].isnan().all()) and bool((got[4][i] == -1).all())
        assert got[0][i] == 0 if i == 7 else got[0][i].isnan()
    assert got[1][0] == -math.inf and got[0][0] == -math.inf and got[2][0] == 0
    assert got[4][0].tolist() == list(range(16)) and bool((got[3][0] == -math.inf).all())


@pytest.mark.parametrize("t,v,ranks", [(400, 700, 1), (64, 2678, 4), (300, 32768, 2), (8, 131072, 3), (1, 20000, 1)])
def test_a_likely_token_keeps_its_digits(worlds, t, v, ranks):
    """All logits but one are equal, so that all their terms are one e, and that one's is 1: s = 1 + (V - 1) e, chosen between
    1.02 and 1.05.  s is off by the three roundings of the eight terms next to the 1, at most 3 U (values below 2), and by
    what is relative to (V - 1) e <= 0.05: e's own error, |y| 3 U + 2 U with |y| <= 15 log2 e, and three roundings, one by
    one below 0.05 (65 + 2 + 3) U = 3.5 U.  Then ln s, a relative 4 U and ln s below 0.05, and one rounding."""
    x = torch.zeros(t, v)
    top = torch.randint(0, v, (t,), generator=torch.Generator().manual_seed(v))
    share = 0.02 + 0.03 * torch.rand(t, generator=torch.Generator().manual_seed(t))
    x[torch.arange(t), top] = ((v - 1) / share).log()
    rows = Rows(x, DT.FP32, ranks, 2)
    lp, lse, entropy, values, ids = rows.run(worlds(ranks), top)
    exact = reference(rows.x, top, 1.0, 2)
    assert bool(((lp - exact[0]).abs() <= 7 * U).all()), float((lp - exact[0]).abs().max() / U)
    assert torch.equal(values[:, 0], lp) and torch.equal(ids[:, 0], top)


@pytest.mark.parametrize("t,v,ranks", [(300, 1000, 1), (64, 4096, 2), (300, 32768, 1), (8, 131072, 3)])
@pytest.mark.parametrize("share", [1e-3, 1e-4, 1e-5, 1e-6])
def test_how_near_a_very_likely_token_comes(worlds, t, v, ranks, share):
    """As above with s - 1 = share: three roundings next to the 1, 3 U, stay however small ln s is.  The others' terms are off
    by what y and their carrying over to a larger maximum are, 3 U of either's exponent, and two exponentials, 2 U each; five
    roundings of their sums; ln s and the result are off by 6 U of themselves."""
    x = torch.zeros(t, v)
    top = torch.randint(0, v, (t,), generator=torch.Generator().manual_seed(v))
    y = ((v - 1) / (share * (0.7 + 0.6 * torch.rand(t, generator=torch.Generator().manual_seed(t))))).log()
    x[torch.arange(t), top] = y
    rows = Rows(x, DT.FP32, ranks, 2)
    lp, lse, entropy, values, ids = rows.run(worlds(ranks), top)
    exact = reference(rows.x, top, 1.0, 2)
    tol = 3 * U + 1.3 * share * (6 * y.double() / math.log(2) + 9) * U + 6 * U * exact[0].abs()
    assert bool(((lp - exact[0]).abs() <= tol).all()), float(((lp - exact[0]).abs() / tol).max())
    assert torch.equal(values[:, 0], lp) and torch.equal(ids[:, 0], top)


@pytest.mark.parametrize("dtype", [DT.FP32, DT.BFP16, DT.FP16])
@pytest.mark.parametrize("t,v,ranks", [(5, 40, 1), (4, 2678, 4), (130, 5001, 2), (300, 9000, 3), (1025, 700, 1), (1, 100000, 1)])
def test_a_certain_token_has_probability_one(worlds, dtype, t, v, ranks):
    """Every other logit lies at least 34 below the largest, so that all of them together add less than 10^5 e^-34 < 2^-32
    to its term of exactly 1, and 0 <= ln s < 2^-32.  The largest one's log probability is then within 2^-32 of 0, that of
    another the difference, rounded as a 32-bit subtraction rounds it (2^-32 is far below half its step), lse the logit
    itself; the entropy is at most ln s plus the sum of |y| e^y, below 2^-32 (1 + 34 + 60)."""
    x = rng_tensor(t + v, t, v, scale=2.0).clamp(-10, 10) - 40
    top = torch.randint(0, v, (t,), generator=torch.Generator().manual_seed(v))
    most = rng_tensor(t, t, scale=0.9).clamp(-3, 3) + 7.3
    x[torch.arange(t), top] = most
    rows = Rows(x, dtype, ranks, 3)
    for tokens in (top, (top + v // 2) % v):
        lp, lse, entropy, values, ids = rows.run(worlds(ranks), tokens)
        m = rows.x.float()[torch.arange(t), top]
        exact = (rows.x.float()[torch.arange(t), tokens] - m).double()
        assert bool((torch.where(exact == 0, (lp <= 0) & (lp > -2.0 ** -32), lp == exact)).all())
        assert torch.equal(lse, m.double())
        assert torch.equal(ids[:, 0], top) and bool(((values[:, 0] <= 0) & (values[:, 0] > -2.0 ** -32)).all())
        assert bool((entropy.abs() <= 2.0 ** -32 * 95).all())


@pytest.mark.parametrize("t,v", [(1030, 8000), (3, 100000)])
def test_many_equal_logits(worlds, t, v):
    """Rows in which far more entries reach the bound on the alternatives than its list holds: few values, one value, and
    columns that fall to one lane of the kernel holding all large values beside a sea of equal ones (the exact search has
    to bisect)."""
    g = torch.Generator().manual_seed(v)
    x = torch.randint(0, 3, (t, v), generator=g).float()
    x[0] = 1.5
    x[1] = 0.0
    lane = (torch.arange(v) // 8) % 256 == 7
    x[1, lane] = 1.0 + torch.arange(int(lane.sum())).float() / 512
    x[2] = torch.arange(v).float() // 3 / 64
    tokens = given(t, v, 1)
    rows = Rows(x, DT.FP32, 1, 32, parts=[(0, v)])
    check_rows(rows, rows.run(worlds(1), tokens), tokens, 1.0)


@pytest.mark.parametrize("t,threads", [(129, 1024), (257, 256)])
def test_more_large_logits_in_one_lane_than_its_list_takes(worlds, t, threads):
    """Columns that one lane of a workgroup reads hold all the large values, rising, beside a row of zeros: the alternatives
    are the last of them, found by bisection.  (The lane map is the kernel's; with another one the case is an easy one.)"""
    v = 4 * threads * 600
    w = worlds(1)
    x = torch.zeros(t, v, device="cuda")
    column = torch.arange(v, device="cuda")
    columns = column[(column // 4) % threads == 7]
    x[0, columns] = 1 + torch.arange(len(columns), device="cuda") / 4096
    x[1, columns] = 1 + torch.arange(len(columns), device="cuda").flip(0) / 4096
    values = torch.zeros(t, 32, device="cuda")
    ids = torch.zeros(t, 32, device="cuda", dtype=torch.int64)
    torch.cuda.synchronize()
    model_ops.token_log_probs(w.comms[0], x, t, 0, v, None, None, data_type=DT.FP32, top_count=32, top_values=values,
                              top_ids=ids, stream=w.stream)
    w.sync()
    assert ids[0].tolist() == columns.flip(0)[:32].tolist()
    assert ids[1].tolist() == columns[:32].tolist()
    assert ids[2].tolist() == list(range(32))
    for row in range(3):
        want = torch.log_softmax(x[row].double(), 0)[ids[row]]
        assert float((values[row].double() - want).abs().max()) <= (terms(v) + 8 + 64) * U


def test_outputs_are_optional_and_each_may_go_elsewhere(worlds):
    x = rng_tensor(3, 40, 999)
    tokens = given(40, 999, 2)
    rows = Rows(x, DT.FP32, 2, 4)
    want = rows.run(worlds(2), tokens)
    w = worlds(2)
    only = torch.full((40,), FILL, device="cuda")
    ids = torch.full((40, 4), 77, device="cuda")
    dev = tokens.cuda()
    torch.cuda.synchronize()
    with hccl_amd.group():      # rank 0 wants the entropy alone and has no tokens, rank 1 the ids alone
        for r, (start, count) in enumerate(rows.parts):
            s = rows.shards[r]
            model_ops.token_log_probs(w.comms[r], s, 40, start, count, dev if r else None, None, data_type=DT.FP32,
                                      row_stride=s.stride(0), entropy=None if r else only, top_count=4,
                                      top_ids=ids if r else None, stream=w.stream)
    w.sync()
    assert torch.equal(only.cpu().double(), want[2]) and torch.equal(ids.cpu(), want[4])


def test_ranks_on_their_own_streams_and_a_shared_workspace_in_turn(worlds):
    w = worlds(3)
    streams = [torch.cuda.Stream() for _ in range(3)]
    size = model_ops.token_log_probs_workspace(2, 50001, 8)
    space = torch.empty(size, dtype=torch.uint8, device="cuda")
    for seed in range(3):
        x = rng_tensor(seed, 2, 50001, scale=2.0)
        tokens = given(2, 50001, seed)
        rows = Rows(x, DT.BFP16, 3, 8)
        check_rows(rows, rows.run(w, tokens, 1.0, streams, space), tokens, 1.0)


# ---- their gradient ----------------------------------------------------------------------------------------------
def grad_case(w, rows, tokens, scale, g, e, h, in_place=False, lse=None, entropy=None, ids=None, tight=False):
    """The gradient of every rank's part, joined, and the numbers it was computed from."""
    _, ref_lse, ref_entropy, _, ref_ids, _ = reference(rows.x, tokens, scale, rows.top)
    lse = (ref_lse if lse is None else lse).float()
    entropy = (ref_entropy if entropy is None else entropy).float()
    ids = ref_ids if ids is None else ids
    dev = lambda a, t=torch.float32: None if a is None else a.to(t).cuda().contiguous()  # noqa: E731
    d_lse, d_entropy, d_g, d_e, d_h = dev(lse), dev(entropy), dev(g), dev(e), dev(h)
    d_ids, d_tokens = dev(ids, TORCH[rows.token_type]), dev(tokens, TORCH[rows.token_type])
    out = []
    for r, (start, count) in enumerate(rows.parts):
        s = rows.shards[r]
        stride = s.stride(0) + 5
        room, d = rows.room(1, stride, count if tight else stride)
        d = s if in_place else d
        torch.cuda.synchronize()
        model_ops.token_log_probs_grad(w.comms[r], s, rows.t, start, count, d_tokens, d_lse, d_g, d, data_type=rows.dtype,
                                       token_type=rows.token_type, row_stride=s.stride(0), grad_row_stride=d.stride(0),
                                       scale=scale, entropy=d_entropy, grad_entropy=d_e, top_count=rows.top, top_ids=d_ids,
                                       grad_top_values=d_h, stream=w.stream)
        w.sync()
        assert bool((d[:, count:] == FILL).all())          # the room between the rows stays
        if not in_place:
            assert float(room[0]) == FILL
        out.append(d[:, :count].cpu())
    return torch.cat(out, 1), lse.double(), entropy.double(), ids


def check_grad(rows, got, lse, entropy, ids, tokens, scale, g, e, h):
    """Against the formula in 64 bits on the same lse and entropy."""
    z = rows.x.double() * float(np.float32(scale))
    log_p = z - lse[:, None]
    p = log_p.exp()
    zero = torch.zeros(rows.t, dtype=torch.float64)
    gd = zero if g is None else torch.where(tokens >= 0, g.float().double(), 0.0)
    ed = zero if e is None else e.float().double()
    hd = torch.zeros(rows.t, 1, dtype=torch.float64) if h is None else torch.where(ids >= 0, h.float().double(), 0.0)
    a = gd + hd.sum(1)
    inner = ed[:, None] * (log_p.clamp(min=-1000) + entropy[:, None])
    d = -p * (a[:, None] + inner)
    pos = torch.zeros_like(d)
    if g is not None:
        at = torch.where((tokens >= 0) & (tokens < rows.v), tokens, 0)
        take = torch.where((tokens >= 0) & (tokens < rows.v), gd, 0.0)
        d.scatter_add_(1, at[:, None], take[:, None])
        pos.scatter_add_(1, at[:, None], take.abs()[:, None])
    if h is not None:
        d.scatter_add_(1, ids.clamp(min=0), hd)
        pos.scatter_add_(1, ids.clamp(min=0), hd.abs())
    f = float(np.float32(scale))
    d, pos = d * f, pos * f
    # p: log p is one rounding of a sum of two terms of |z| and |lse|, then two more of its own size and an exponential (2 U)
    # the sums a and (log p + H) e + a: up to 34 and 3 roundings of their terms
    absolute = p * f * (gd.abs()[:, None] + hd.abs().sum(1)[:, None] + ed.abs()[:, None] *
                        (log_p.clamp(min=-1000).abs() + entropy.abs()[:, None]))
    near = torch.where(log_p > -200, z.abs().clamp(max=1e30) + lse.abs()[:, None] + 3 * log_p.abs(), 0.0)
    eps = torch.finfo(TORCH[rows.dtype]).eps
    tiny = torch.finfo(TORCH[rows.dtype]).smallest_normal * eps      # half a step of the smallest values, and flushed ones
    tol = absolute * (near + 44) * U + pos * 36 * U + tiny + 2.0 ** -126
    tol = tol + eps / 2 * (d.abs() + tol) if rows.dtype != DT.FP32 else tol + 2 * U * d.abs()
    off = (got.double() - d).abs()
    assert bool((off <= tol).all()), float((off / tol).max())


GRADS = ["g", "ge", "geh", "h", "e"]


@pytest.mark.parametrize("dtype", [DT.FP32, DT.BFP16, DT.FP16])
@pytest.mark.parametrize("t,v,ranks,which", [
    (1, 1, 1, "geh"), (1, 8, 1, "g"), (3, 9, 2, "geh"), (4, 257, 3, "ge"), (7, 8191, 1, "geh"), (2, 8193, 2, "e"),
    (5, 40001, 3, "geh"), (33, 4096, 2, "h"), (1, 131072, 8, "geh"), (300, 50, 1, "ge")])
def test_gradient(worlds, dtype, t, v, ranks, which):
    x = rng_tensor(t + v, t, v, scale=2.0)
    x[:, v // 3] += 5.0
    tokens = given(t, v, 8)
    top = min(v, 8)
    scale = (1.0, 0.5, 1.5)[(t + v) % 3]
    g = rng_tensor(1, t) if "g" in which else None
    e = rng_tensor(2, t) if "e" in which else None
    h = rng_tensor(3, t, top) if "h" in which else None
    rows = Rows(x, dtype, ranks, top, DT.INT32 if t % 2 else DT.INT64)
    got, lse, entropy, ids = grad_case(worlds(ranks), rows, tokens, scale, g, e, h)
    check_grad(rows, got, lse, entropy, ids, tokens, scale, g, e, h)


@pytest.mark.parametrize("dtype", [DT.FP32, DT.BFP16])
def test_gradient_in_place_equals_the_one_apart(worlds, dtype):
    x = rng_tensor(9, 6, 20011)
    tokens = given(6, 20011, 8)
    g, e, h = rng_tensor(1, 6), rng_tensor(2, 6), rng_tensor(3, 6, 8)
    rows = Rows(x, dtype, 2, 8)
    apart = grad_case(worlds(2), rows, tokens, 1.0, g, e, h)[0]
    assert torch.equal(grad_case(worlds(2), rows, tokens, 1.0, g, e, h, in_place=True)[0], apart)


def test_gradient_with_the_same_index_many_times(worlds):
    """The token among the alternatives, an id that comes twice, ids that were never found (-1) and one beyond V."""
    x = rng_tensor(4, 5, 3001)
    tokens = torch.tensor([7, 3000, 0, -100, 9])
    ids = torch.tensor([[7, 7, 7, 8], [3000, 0, 3000, 1], [-1, 0, 5, -1], [2, 2, 1, 2], [9, 9, 8, 9]])
    g, e, h = rng_tensor(1, 5), rng_tensor(2, 5), rng_tensor(3, 5, 4)
    rows = Rows(x, DT.FP32, 3, 4)
    got, lse, entropy, _ = grad_case(worlds(3), rows, tokens, 1.0, g, e, h, ids=ids)
    check_grad(rows, got, lse, entropy, ids, tokens, 1.0, g, e, h)


@pytest.mark.parametrize("dtype", [DT.FP32, DT.BFP16, DT.FP16])
def test_gradient_of_masked_rows(worlds, dtype):
    x = rng_tensor(2, 8, 9001, scale=2.0)
    low = torch.finfo(TORCH[dtype]).min
    x[0] = -math.inf
    x[1, ::2] = -math.inf
    x[2, 10:] = low
    x[3] = -math.inf
    x[3, 4000] = 1.0
    x[5] = math.nan                 # a row that carries no gradient is not read
    tokens = torch.tensor([5, 7, 3, 4000, 1, -100, 2, 2])
    g = torch.tensor([1.0, 2.0, -1.0, 0.5, 0.0, 3.0, 1.0, 1.0])
    e = torch.tensor([1.0, 1.0, 1.0, 1.0, 0.0, 0.0, 0.0, -2.0])
    rows = Rows(x, dtype, 2, 0)
    got, lse, entropy, ids = grad_case(worlds(2), rows, tokens, 1.0, g, e, None)
    for i in (0, 4, 5):
        assert bool((got[i] == 0).all()), i
    keep = [1, 2, 3, 6, 7]
    part = Rows(x[keep], dtype, 2, 0)
    check_grad(part, got[keep], lse[keep], entropy[keep], None, tokens[keep], 1.0, g[keep], e[keep], None)
    if dtype != DT.FP16:            # a row of the lowest value alone counts as masked (fp16's is an ordinary number)
        lowest = Rows(torch.full((1, 100), low), dtype, 1, 0)
        one = torch.ones(1)
        assert bool((grad_case(worlds(1), lowest, torch.tensor([3]), 1.0, one, one, None)[0] == 0).all())


@pytest.mark.parametrize("most", [5.0, 20.0, 40.0, 60.0, 1000.0, -300.0])
@pytest.mark.parametrize("share", [1e-2, 1e-5])
def test_gradient_of_likely_tokens_after_the_forward_pass(worlds, most, share):
    """Forward, then backward with what it left, against the gradient in 64 bits, at a large log-sum-exp and 1 - p = share.  The
    backward pass takes log p from the 32-bit lse: that is off by one rounding of |lse| U and by the forward pass's ln s, 3 U
    and 6 U of itself; log p takes one rounding more, its way to p two and an exponential 2 U.  p is off by that share of
    itself: beside a p near 1, 1 - p has no more digits than |lse| U leaves it.  The sum with the one-hot term and the
    products take four roundings."""
    t, v, ranks = 40, 4096, 2
    top = torch.randint(0, v, (t,), generator=torch.Generator().manual_seed(5))
    wide = share * (0.7 + 0.6 * torch.rand(t, generator=torch.Generator().manual_seed(6)))
    x = (most - ((v - 1) / wide).log())[:, None].expand(t, v).clone()
    x[torch.arange(t), top] = most
    g = rng_tensor(8, t)
    w = worlds(ranks)
    rows = Rows(x, DT.FP32, ranks)
    _, lse, entropy, _, _ = rows.run(w, top)
    got = grad_case(w, rows, top, 1.0, g, None, None, lse=lse, entropy=entropy)[0].double()
    log_p = reference(rows.x, top, 1.0, 0)[5]
    p, gd = log_p.exp(), g.double()[:, None]
    exact = -p * gd
    exact.scatter_add_(1, top[:, None], gd)
    off = p * (abs(most) + 3 + 6 * share + 3 * log_p.abs() + 2) * U
    assert bool(((got - exact).abs() <= (off + 4 * U * p) * gd.abs() + 4 * U * exact.abs()).all())


def test_gradient_against_differences_of_the_forward_pass(worlds):
    """Central differences of the framework's own forward pass along random directions.  The loss is a sum of 4 log
    probabilities, 4 entropies and 8 alternatives with weights up to 3: every one is off by at most 400 U (V = 501), so a
    difference over 2 h = 2^-5 by 16 * 3 * 400 U * 2 / 2^-5 < 0.08 at the very worst; the third derivative along a unit
    direction adds h^2 / 6 * (a few) < 0.001.  Directions are scaled so that the derivative is of the order of ten."""
    t, v, top = 4, 501, 2
    x = rng_tensor(11, t, v)
    tokens = given(t, v, 4)
    g, e, h = rng_tensor(1, t), rng_tensor(2, t), rng_tensor(3, t, top)
    w = worlds(2)
    rows = Rows(x, DT.FP32, 2, top)
    base = rows.run(w, tokens)
    got, _, _, ids = grad_case(w, rows, tokens, 1.0, g, e, h, lse=base[1], entropy=base[2], ids=base[4])

    def loss(y):
        lp, _, ent, values, got_ids = Rows(y, DT.FP32, 2, top).run(w, tokens)
        assert torch.equal(got_ids, ids)
        return float((torch.where(tokens >= 0, g.double(), 0.0) * lp).sum() + (e.double() * ent).sum() +
                     (h.double() * values).sum())
    step = 2.0 ** -6
    for seed in range(4):
        u = rng_tensor(20 + seed, t, v)
        u = u + 2 * torch.sign(got)                       # lies along the gradient, so that the derivative is not small
        u = u / u.norm() * math.sqrt(t)
        # the perturbation must not reorder the alternatives: they are pinned by a gap much larger than the step
        numeric = (loss(x + step * u) - loss(x - step * u)) / (2 * step)
        analytic = float((got.double() * u.double()).sum())
        assert abs(numeric - analytic) <= 0.08 + 0.02 * abs(analytic), (numeric, analytic)


# ---- gradient norm -------------------------------------------------------------------------------------------------
def norm_case(w, per_rank, max_norm=1.0, scale=1.0, behind=9):
    """per_rank: lists of (host tensor, type, element offset); returns every rank's (norm, factor)."""
    keep, descr = [], []
    for tensors in per_rank:
        mine = []
        for x, dtype, offset in tensors:
            room = torch.full((offset + x.numel() + behind,), 1e4, dtype=TORCH[dtype], device="cuda")
            room[offset:offset + x.numel()] = x.to(TORCH[dtype]).cuda()
            keep.append(room)
            mine.append((room[offset:], x.numel(), dtype))
        descr.append(mine)
    n = len(per_rank)
    size = model_ops.grad_norm_workspace(sum(len(d) for d in descr))
    space = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
    out = torch.full((n, 3), FILL, device="cuda")
    torch.cuda.synchronize()
    with hccl_amd.group():
        for r in range(n):
            model_ops.grad_norm(w.comms[r], descr[r], max_norm, out[r], scale=scale, workspace=space, workspace_bytes=size,
                                stream=w.stream)
    w.sync()
    assert bool((out[:, 2] == FILL).all())
    assert torch.equal(out.nan_to_num(9e9), out[:1].expand(n, 3).nan_to_num(9e9))
    return out[0, :2].cpu().double()


def norm_reference(per_rank, max_norm, scale):
    total = sum(float(x.to(TORCH[dtype]).double().square().sum()) for tensors in per_rank for x, dtype, _ in tensors)
    norm = abs(scale) * math.sqrt(total)
    return norm, scale * (min(1.0, max_norm / (norm + 1e-6)) if max_norm > 0 else 1.0)


@pytest.mark.parametrize("dtype", [DT.FP32, DT.BFP16, DT.FP16])
@pytest.mark.parametrize("sizes", [[1], [0, 7], [8191, 8192, 8193], [4095, 4096, 4097, 0, 1, 3], [1 << 20, 100003]])
@pytest.mark.parametrize("ranks", [1, 3])
def test_norm(worlds, dtype, sizes, ranks):
    per_rank = [[(rng_tensor(10 * r + i, n), dtype, (i + r) % 3) for i, n in enumerate(sizes)] for r in range(ranks)]
    for max_norm, scale in ((1.0, 1.0), (1e9, 0.25), (0.0, -2.0)):
        got = norm_case(worlds(ranks), per_rank, max_norm, scale)
        norm, factor = norm_reference(per_rank, max_norm, scale)
        # 64-bit sums of at most 2^21 terms are off by 2^-32 at the very worst; then one rounding to 32 bits
        assert abs(got[0] - norm) <= (U + 2.0 ** -32) * norm + 1e-45
        assert abs(got[1] - factor) <= (U + 2.0 ** -31) * abs(factor)


def test_norm_of_many_tensors_of_all_types_and_ranks_without_any(worlds):
    types = [DT.FP32, DT.BFP16, DT.FP16]
    many = [(rng_tensor(i, 1 + (i * 37) % 500), types[i % 3], i % 2) for i in range(533)]
    per_rank = [many[:500], [], many[500:]]
    norm, factor = norm_reference(per_rank, 2.0, 1.0)
    got = norm_case(worlds(3), per_rank, 2.0, 1.0)
    assert abs(got[0] - norm) <= 2 * U * norm and abs(got[1] - factor) <= 2 * U * factor
    assert norm_case(worlds(3), [[], [], []], 1.0, 0.5).tolist() == [0.0, 0.5]


def test_norm_keeps_what_32_bits_would_lose(worlds):
    for value in (1e30, 1e-30):
        got = norm_case(worlds(1), [[(torch.full((1000,), value), DT.FP32, 0)]], 0.0, 1.0)
        want = float(np.float32(value)) * math.sqrt(1000)
        assert abs(got[0] - want) <= 2 * U * want
    for bad in (math.nan, math.inf):
        x = torch.ones(5000)
        x[4321] = bad
        got = norm_case(worlds(2), [[(x, DT.BFP16, 1)], [(torch.ones(3), DT.FP32, 0)]])
        assert not math.isfinite(got[0])


def test_norm_is_the_same_every_time(worlds):
    per_rank = [[(rng_tensor(r, 300001), DT.FP32, 0)] for r in range(3)]
    first = norm_case(worlds(3), per_rank)
    for _ in range(3):
        assert torch.equal(norm_case(worlds(3), per_rank), first)


@pytest.mark.parametrize("dtype", [DT.FP32, DT.BFP16, DT.FP16])
def test_memory_that_ends_with_the_last_element(worlds, dtype):
    """No byte behind a buffer is read or written either: the run of this test on the CPU (test_emulated_model_ops.py) looks
    at every access."""
    for t, v, ranks in ((1, 1, 1), (2, 7, 1), (3, 9, 3), (2, 2055, 2), (5, 8193, 1), (1, 40003, 3), (260, 300, 2)):
        for offset in (0, 1):
            x = rng_tensor(t + v, t, v)
            tokens, top = given(t, v, 1), min(v, 5)
            g, e, h = rng_tensor(1, t), rng_tensor(2, t), rng_tensor(3, t, top)
            rows = Rows(x, dtype, ranks, top, pad=offset, offset=offset, tight=True)
            check_rows(rows, rows.run(worlds(ranks), tokens), tokens, 1.0)
            got, lse, entropy, ids = grad_case(worlds(ranks), rows, tokens, 1.0, g, e, h, tight=True)
            check_grad(rows, got, lse, entropy, ids, tokens, 1.0, g, e, h)
    per_rank = [[(rng_tensor(n, n), dtype, n % 3) for n in (1, 3, 8, 15, 8191, 8193)]]
    norm, factor = norm_reference(per_rank, 1.0, 1.0)
    got = norm_case(worlds(1), per_rank, behind=0)
    assert abs(got[0] - norm) <= 2 * U * norm and abs(got[1] - factor) <= 2 * U * factor
    for fp8 in (False, True):
        for combo in [c for c in COMBOS if c[1] == dtype]:
            run_adamw(worlds(1), [Tensor(n, combo, fp8, n, n % 3, behind=0) for n in (1, 3, 257, 1023, 4099)], fp8)


# ---- AdamW -----------------------------------------------------------------------------------------------------------
E4M3 = torch.float8_e4m3fn
COMBOS = [(DT.FP32, DT.FP32, False), (DT.FP32, DT.BFP16, False), (DT.FP32, DT.FP16, False), (DT.BFP16, DT.BFP16, False),
          (DT.BFP16, DT.BFP16, True), (DT.BFP16, DT.FP32, True), (DT.BFP16, DT.FP32, False), (DT.FP16, DT.FP16, True),
          (DT.FP16, DT.FP16, False), (DT.FP16, DT.FP32, True), (DT.FP16, DT.FP32, False)]


class Tensor:
    """One tensor's buffers, each at an element offset inside a larger one that has to stay as it was."""

    def __init__(self, n, combo, fp8, seed, offset=0, fresh=False, behind=8):
        self.behind, self.n, (self.param_type, self.grad_type, self.with_master), self.fp8 = behind, n, combo, fp8
        self.rooms = {}
        blocks = -(-n // 256)
        w = rng_tensor(seed, n, scale=0.05)
        g = rng_tensor(seed + 1, n, scale=0.01)
        g[:n // 7] = 0
        if n > 600:
            g[256:512] = 0
        self.place("param", w.to(TORCH[self.param_type]), offset)
        self.place("grad", g.to(TORCH[self.grad_type]), offset)
        if self.with_master:
            self.place("master", w, offset)
        m = rng_tensor(seed + 2, n, scale=0.002) * (0 if fresh else 1)
        root = (m.abs() * 3 + 1e-4) * (0 if fresh else 1)
        if n > 600 and not fresh:
            m[256:512] = 0
            root[256:512] = 0
        if fp8:
            for name, x in (("exp_avg", m), ("exp_avg_sq", root)):
                pad = torch.zeros(blocks * 256)
                pad[:n] = x
                most = pad.view(-1, 256).abs().amax(1)
                unit = torch.where(most > 0, 448 / most, 0.0)
                code = (pad.view(-1, 256) * unit[:, None]).to(E4M3).view(-1)[:n]
                self.place(name, code.view(torch.uint8), offset)
                self.place(name + "_scale", most / 448, 0)
        else:
            self.place("exp_avg", m, offset)
            self.place("exp_avg_sq", root.square(), offset)

    def place(self, name, x, offset):
        room = torch.full((offset + x.numel() + self.behind,), 77, dtype=x.dtype, device="cuda")
        room[offset:offset + x.numel()] = x.cuda()
        self.rooms[name] = (room, offset, x.numel())

    def view(self, name):
        room, offset, n = self.rooms[name]
        return room[offset:offset + n]

    def descr(self):
        d = {k: self.rooms[k][0][self.rooms[k][1]:] for k in self.rooms}
        return dict(d, count=self.n, param_type=self.param_type, grad_type=self.grad_type)

    def host(self):
        return {k: self.view(k).cpu().clone() for k in self.rooms}

    def untouched_around(self):
        for name, (room, offset, n) in self.rooms.items():
            assert bool((room[:offset] == 77).all()) and bool((room[offset + n:] == 77).all()), name


def wide(codes, scales):
    return codes.view(E4M3).double() * scales.double().repeat_interleave(256)[:codes.numel()]


def check_adamw(t, before, step, lr, beta1, beta2, eps, decay, clip):
    """The definition in 64 bits.  The hyper-parameters are rounded to 32 bits on the way into the kernel (U each)."""
    t.untouched_around()
    after = t.host()
    assert torch.equal(after["grad"], before["grad"])
    w = (before["master"] if t.with_master else before["param"]).double()
    g = before["grad"].double() * clip
    if t.fp8:
        m, v = wide(before["exp_avg"], before["exp_avg_scale"]), wide(before["exp_avg_sq"], before["exp_avg_sq_scale"]) ** 2
    else:
        m, v = before["exp_avg"].double(), before["exp_avg_sq"].double()
    size_m = (beta1 * m).abs() + ((1 - beta1) * g).abs()
    m = beta1 * m + (1 - beta1) * g
    v = beta2 * v + (1 - beta2) * g * g
    denominator = v.sqrt() / math.sqrt(1 - beta2 ** step) + eps
    update = lr / (1 - beta1 ** step) * m / denominator
    new = w * (1 - lr * decay) - update
    # m: eight roundings (decoding, clip, factors, sum); v: the same plus the squares'; its root half of that
    tol_m, tol_v = 8 * U * size_m, 12 * U * v
    # the step: m's, the root's (6 + 2 for the instruction's 1 ulp), the denominator's, the reciprocal's, the factors'
    tol_w = 24 * U * lr / (1 - beta1 ** step) * (size_m / denominator) + 4 * U * w.abs() + 2.0 ** -126
    if t.with_master:
        assert bool(((after["master"].double() - new).abs() <= tol_w).all())
        assert torch.equal(after["param"], after["master"].to(TORCH[t.param_type]))
    else:
        kind = torch.finfo(TORCH[t.param_type])
        half = 0 if t.param_type == DT.FP32 else kind.eps / 2
        tol = tol_w + half * (new.abs() + tol_w) + (kind.smallest_normal * kind.eps if half else 0)
        assert bool(((after["param"].double() - new).abs() <= tol).all())
    if not t.fp8:
        assert bool(((after["exp_avg"].double() - m).abs() <= tol_m + 1e-44).all())
        assert bool(((after["exp_avg_sq"].double() - v).abs() <= tol_v + 1e-37).all())
        return
    pad = -t.n % 256
    for name, x, tol in (("exp_avg", m, tol_m), ("exp_avg_sq", v.sqrt(), 8 * U * v.sqrt())):
        scale = after[name + "_scale"].double()
        most = torch.nn.functional.pad(x.abs(), (0, pad)).view(-1, 256).amax(1)
        far = torch.nn.functional.pad(tol, (0, pad)).view(-1, 256).amax(1) + 2 * U * most
        assert bool(((scale * 448 - most).abs() <= far + 1e-37).all()), name
        got = wide(after[name], after[name + "_scale"])
        unit = scale.repeat_interleave(256)[:t.n]
        # half a step of e4m3: 2^-4 of the value, at least 2^-10 of the scale; a root above 0 is at least a whole 2^-9
        least = 2.0 ** -10 if name == "exp_avg" else 2.0 ** -9
        allowed = torch.maximum(x.abs() * 2.0 ** -4, unit * least) * (1 + 1e-5) + 2 * tol
        assert bool(((got - x).abs() <= allowed + 1e-37).all()), name
    root = wide(after["exp_avg_sq"], after["exp_avg_sq_scale"])
    assert bool(((root > 0) == (v > 0)).all())


def run_adamw(w, tensors, fp8, step=1000, lr=1e-2, beta1=0.9, beta2=0.99, eps=1e-8, decay=0.1, clip=None, check=True, **k):
    before = [t.host() for t in tensors]
    factor = torch.tensor([3.0, clip], device="cuda") if clip is not None else None
    torch.cuda.synchronize()
    model_ops.adamw(w.comms[0], [t.descr() for t in tensors], step, lr, beta1, beta2, eps, decay,
                    DT.FP8E4M3 if fp8 else DT.FP32, clip=factor, stream=w.stream, **k)
    w.sync()
    if check:
        for t, b in zip(tensors, before):
            check_adamw(t, b, step, lr, beta1, beta2, eps, decay, clip if clip is not None else 1.0)
    return before


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("combo", COMBOS)
def test_adamw(worlds, combo, fp8):
    sizes = [1, 7, 8, 255, 256, 257, 1000, 4095, 4096, 4097, 10007, 0]
    for step, clip, offset in ((1, None, 0), (1000, 0.37, 1), (3, 0.5, 3)):
        tensors = [Tensor(n, combo, fp8, 10 * i + step, offset, fresh=step == 1) for i, n in enumerate(sizes)]
        run_adamw(worlds(1), tensors, fp8, step=step, clip=clip)


@pytest.mark.parametrize("fp8", [False, True])
def test_adamw_over_many_tensors_of_all_kinds(worlds, fp8):
    tensors = [Tensor(1 + (97 * i) % 1500, COMBOS[i % len(COMBOS)], fp8, i, i % 4) for i in range(311)]
    run_adamw(worlds(1), tensors, fp8, clip=0.8)


@pytest.mark.parametrize("fp8", [False, True])
def test_adamw_with_its_step_and_rate_on_the_device(worlds, fp8):
    """A captured step reads both when it runs.  The factors are then formed in 32 bits: 1 - beta^n = -expm1(n ln beta) is
    off by 4 U plus the U of ln beta times n |ln beta| beta^n / (1 - beta^n) < 1: inside the eight roundings allowed for the
    factors."""
    w = worlds(1)
    for step in (1, 2, 77, 100000):
        tensors = [Tensor(5000, (DT.BFP16, DT.BFP16, True), fp8, step, 0, fresh=step == 1)]
        on_device = torch.tensor([step], dtype=torch.int64, device="cuda")
        rate = torch.tensor([1e-2], device="cuda")
        before = run_adamw(w, tensors, fp8, step=12345, lr=5.0, check=False, step_on_device=on_device, lr_on_device=rate)
        check_adamw(tensors[0], before[0], step, float(rate), 0.9, 0.99, 1e-8, 0.1, 1.0)


def test_adamw_skips_a_step_whose_norm_is_not_finite(worlds):
    w = worlds(1)
    for bad in (math.nan, math.inf):
        t = Tensor(5000, (DT.BFP16, DT.BFP16, True), False, 3)
        before = t.host()
        factor = torch.tensor([bad, 0.5], device="cuda")
        torch.cuda.synchronize()
        model_ops.adamw(w.comms[0], [t.descr()], 5, 1e-2, clip=factor, skip_non_finite=True, stream=w.stream)
        w.sync()
        after = t.host()
        assert all(torch.equal(after[k], before[k]) for k in before)
        model_ops.adamw(w.comms[0], [t.descr()], 5, 1e-2, clip=factor, stream=w.stream)
        w.sync()
        assert not torch.equal(t.host()["master"], before["master"])


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("eps", [0.0, 1e-30, 2.0 ** -126, 1e-8])
def test_adamw_with_second_moments_below_the_smallest_normal_number(worlds, fp8, eps):
    """Gradients so small that v = (1 - beta2) g^2 is subnormal: half a step is then 2^-150, and relative to v
    2^-150 / v, of which the root, and with it the step m / root, takes half.  (One block of equal elements: an FP8 state's
    code is the largest one, so that the unrounded step is what is looked at.)  The other roundings of the step are fewer
    than 24, each U of it; 2^-126 stands for results that are subnormal themselves."""
    n, beta1, beta2, lr = 256, 0.9, 0.999, 1.0
    for exponent in (-59, -61, -64, -67):
        t = Tensor(n, (DT.FP32, DT.FP32, False), fp8, 1, fresh=True)
        t.view("param").zero_()
        g = torch.full((n,), 1.5 * 2.0 ** exponent)
        t.view("grad").copy_(g)
        run_adamw(worlds(1), [t], fp8, 1, lr, beta1, beta2, eps, 0.0, check=False)
        v = (1 - beta2) * g.double() ** 2
        assert 2.0 ** -148 < float(v[0]) < 2.0 ** -126
        update = lr * g.double() / (g.double().abs() + eps)
        assert bool(((t.view("param").cpu().double() + update).abs() <= (24 * U + 2.0 ** -150 / v) * update + 2.0 ** -126).all())


@pytest.mark.parametrize("fp8", [False, True])
def test_adamw_states_are_the_bits_of_elementwise_operations(worlds, fp8):
    """m and v, or their codes and scales, over five steps: every product, sum, root and quotient rounded to 32 bits."""
    n, beta1, beta2 = 256 * 1200 + 77, 0.9, 0.99
    t = Tensor(n, (DT.BFP16, DT.BFP16, True), fp8, 11)
    f = lambda x: torch.tensor(x, dtype=torch.float32)  # noqa: E731
    host = t.host()
    m, v = host["exp_avg"], host["exp_avg_sq"]
    units = lambda x: x.repeat_interleave(256)[:n]  # noqa: E731
    blocks = lambda x: torch.nn.functional.pad(x, (0, -n % 256)).view(-1, 256).abs().amax(1)  # noqa: E731
    if fp8:
        m, m_scale = m.view(E4M3).float(), host["exp_avg_scale"]
        v, v_scale = v.view(E4M3).float(), host["exp_avg_sq_scale"]
    for step in range(1, 6):
        t.view("grad").copy_(rng_tensor(step, n, scale=0.01).to(torch.bfloat16))
        g = t.host()["grad"].float() * f(0.37)
        if fp8:
            m, v = m * units(m_scale), (v * units(v_scale)).square()
        m = m * f(beta1) + g * f(1 - beta1)
        v = v * f(beta2) + g * g * f(1 - beta2)
        run_adamw(worlds(1), [t], fp8, step=step, clip=0.37, check=False)
        got = t.host()
        if fp8:
            root = v.double().sqrt().float()      # (rounds as the root in 32 bits: 53 bits are more than twice 24 and two)
            most, most_root = blocks(m), blocks(root)
            m_scale, v_scale = most * f(448.0).reciprocal(), most_root * f(448.0).reciprocal()
            m = (m * units(most.reciprocal() * 448)).to(E4M3)
            v = torch.where(root > 0, (root * units(most_root.reciprocal() * 448)).clamp(min=2.0 ** -9), 0.0).to(E4M3)
            assert torch.equal(got["exp_avg_scale"], m_scale) and torch.equal(got["exp_avg_sq_scale"], v_scale), step
            assert torch.equal(got["exp_avg"], m.view(torch.uint8)) and torch.equal(got["exp_avg_sq"], v.view(torch.uint8)), step
            m, v = m.float(), v.float()
        else:
            assert torch.equal(got["exp_avg"], m) and torch.equal(got["exp_avg_sq"], v), step


def test_adamw_quantises_as_the_type_says(worlds):
    """Codes of a block whose largest magnitude is 448 / 0.1: exactly the nearest e4m3 values, subnormal ones among them."""
    n = 4096
    t = Tensor(n, (DT.FP32, DT.FP32, False), True, 1, fresh=True)
    g = rng_tensor(5, n) * torch.exp2(torch.arange(n).float() % 20 - 17)
    g[::256] = 448.0
    t.view("grad").copy_(g)
    run_adamw(worlds(1), [t], True, step=1, beta1=0.0, beta2=0.0)
    got = t.host()
    scale = got["exp_avg_scale"].repeat_interleave(256)
    assert bool((scale == g.view(-1, 256).abs().amax(1).repeat_interleave(256) * torch.tensor(448.0).reciprocal()).all())
    clean = g.view(-1, 256).abs().amax(1).repeat_interleave(256) == 448.0
    want = g.to(E4M3).view(torch.uint8)
    assert torch.equal(got["exp_avg"][clean], want[clean])


# ---- beyond 32 bits -----------------------------------------------------------------------------------------------------
def test_logits_beyond_32_bits_of_elements(worlds):
    """2^32 logits and a few rows more, in place: the last rows lie beyond every 32-bit offset."""
    v, t = 131072, (1 << 15) + 5
    w = worlds(1)
    x = torch.zeros(t, v, dtype=torch.bfloat16, device="cuda")
    tail = (rng_tensor(3, 6, v) * 2).to(torch.bfloat16)
    x[-6:] = tail.cuda()
    tokens = torch.full((t,), 11, device="cuda")
    tokens[:-6] = -100
    lp, lse, ent = (torch.full((t,), FILL, device="cuda") for _ in range(3))
    ids = torch.zeros(t, 3, dtype=torch.int64, device="cuda")
    values = torch.zeros(t, 3, device="cuda")
    g = torch.full((t,), 0.5, device="cuda")
    torch.cuda.synchronize()
    model_ops.token_log_probs(w.comms[0], x, t, 0, v, tokens, lp, data_type=DT.BFP16, lse=lse, entropy=ent, top_count=3, top_values=values,
                              top_ids=ids, stream=w.stream)
    model_ops.token_log_probs_grad(w.comms[0], x, t, 0, v, tokens, lse, g, x, data_type=DT.BFP16, entropy=ent,
                                   grad_entropy=g, stream=w.stream)
    w.sync()
    rows = Rows(tail, DT.BFP16, 1, 3, parts=[(0, v)])
    got = tuple(a[-6:].cpu().double() for a in (lp, lse, ent, values)) + (ids[-6:].cpu(),)
    eleven = torch.full((6,), 11)
    check_rows(rows, got, eleven, 1.0)
    check_grad(rows, x[-6:].cpu(), got[1], got[2], None, eleven, 1.0, g[-6:].cpu(), g[-6:].cpu(), None)
    # rows of zeros: uniform, whose entropy has no gradient beyond rounding
    assert abs(float(lse[7]) - math.log(v)) < 1e-5 and lp[7] == 0 and ids[7].tolist() == [0, 1, 2]
    assert float(x[:8].float().abs().max()) < 1e-9


def test_more_rows_than_a_launch_of_the_gradient_takes(worlds):
    """2^23 + 5 rows of three logits, about the most a call may have: all of them against torch in 64 bits, on the GPU.
    s <= 3 has a handful of roundings, log p and the gradient a few more: 16 U of the largest terms, |z| <= 20 and 20."""
    t, v, top = (1 << 23) + 5, 3, 2
    w = worlds(1)
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(t, v, device="cuda", generator=g).mul_(3).clamp_(-10, 10)
    tokens = torch.randint(0, v, (t,), device="cuda", dtype=torch.int32, generator=g)
    lp, lse, entropy, ge = (torch.full((t + 1,), FILL, device="cuda") for _ in range(4))
    values = torch.full((t + 1, top), FILL, device="cuda")
    ids = torch.full((t + 1, top), 77, device="cuda", dtype=torch.int32)
    d = torch.full((t + 1, v), FILL, device="cuda")
    ge.normal_(generator=g).clamp_(-4, 4)
    torch.cuda.synchronize()
    model_ops.token_log_probs(w.comms[0], x, t, 0, v, tokens, lp, token_type=DT.INT32, lse=lse, entropy=entropy, top_count=top,
                              top_values=values, top_ids=ids, stream=w.stream)
    model_ops.token_log_probs_grad(w.comms[0], x, t, 0, v, tokens, lse, ge, d, token_type=DT.INT32, entropy=entropy,
                                   grad_entropy=ge, top_count=top, top_ids=ids, grad_top_values=values, stream=w.stream)
    w.sync()
    for a in (lp, lse, entropy, values[:, 0], values[:, 1], d[:, 0], d[:, 2]):
        assert float(a[-1]) == FILL
    log_p = torch.log_softmax(x.double(), 1)
    at = tokens.long()[:, None]
    close = lambda a, b, bound: float((a[:t].double() - b).abs().max()) <= 16 * U * bound  # noqa: E731
    assert close(lp, log_p.gather(1, at)[:, 0], 20) and close(lse, torch.logsumexp(x.double(), 1), 20)
    assert close(entropy, -(log_p.exp() * log_p).sum(1), 20)
    order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(ids[:t].long(), order) and close(values, log_p.gather(1, order), 20)
    gd, hd = ge[:t].double(), values[:t].double()
    p = log_p.exp()
    want = -p * (gd + hd.sum(1))[:, None] - gd[:, None] * p * (log_p + entropy[:t].double()[:, None])
    want.scatter_add_(1, at, gd[:, None]).scatter_add_(1, order, hd)
    assert close(d, want, 20 * 64)       # terms of up to 4 + 40 + 4 (20 + 2), each p 20 U off


def test_tensors_beyond_32_bits_of_elements(worlds):
    n, tail = (1 << 32) + 1000, 3000
    w = worlds(1)
    param = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    grad = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    m = torch.zeros(n, dtype=torch.uint8, device="cuda")
    v = torch.zeros(n, dtype=torch.uint8, device="cuda")
    m_scale, v_scale = (torch.zeros(-(-n // 256), device="cuda") for _ in range(2))
    weights, g = (rng_tensor(5, tail, scale=0.1)).to(torch.bfloat16), (rng_tensor(6, tail, scale=0.1)).to(torch.bfloat16)
    param[-tail:], grad[-tail:] = weights.cuda(), g.cuda()
    result = torch.zeros(2, device="cuda")
    space = torch.empty(model_ops.grad_norm_workspace(1), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    model_ops.grad_norm(w.comms[0], [(grad, n, DT.BFP16)], 0.0, result, workspace=space, workspace_bytes=space.numel(),
                        stream=w.stream)
    model_ops.adamw(w.comms[0], [dict(param=param, grad=grad, exp_avg=m, exp_avg_sq=v, exp_avg_scale=m_scale,
                                      exp_avg_sq_scale=v_scale, count=n, param_type=DT.BFP16, grad_type=DT.BFP16)],
                    1, 1e-2, 0.9, 0.99, 1e-8, 0.1, DT.FP8E4M3, clip=result, stream=w.stream)
    w.sync()
    norm = float(g.double().square().sum().sqrt())
    assert abs(float(result[0]) - norm) <= 2 * U * norm and float(result[1]) == 1.0
    update = 1e-2 * g.double() / (g.double().abs() + 1e-8)         # the first step's m / sqrt(v) is the gradient's sign
    want = weights.double() * (1 - 1e-3) - update
    assert bool(((param[-tail:].cpu().double() - want).abs() <= 2.0 ** -8 * want.abs() + 64 * U * 1e-2).all())
    last = -(-n // 256) - 1
    assert float(m_scale[last]) > 0 and float(m_scale[0]) == 0 and not bool(param[:-tail].any())
    codes = wide(m[last * 256:].cpu(), m_scale[last:].cpu())
    near = 0.1 * g.double()[-codes.numel():]
    assert bool(((codes - near).abs() <= torch.maximum(near.abs() * 2.0 ** -4, m_scale[last].cpu().double() * 2.0 ** -10) * 1.001).all())


# ---- together ---------------------------------------------------------------------------------------------------------
def test_calls_can_be_captured_into_a_graph_and_replayed(worlds):
    """The log probabilities in both forms (rows that share workgroups and rows that do not), their gradient, the norm and
    a step whose number lives on the device: every replay equals the eager call on the same state."""
    w = worlds(2)
    few, many = Rows(rng_tensor(1, 3, 50001), DT.BFP16, 2, 8), Rows(rng_tensor(2, 1100, 300), DT.FP32, 2, 4)
    few_tokens, many_tokens = given(3, 50001, 1).cuda(), given(1100, 300, 2).cuda()
    size = model_ops.token_log_probs_workspace(3, 50001, 8)
    space = torch.empty(size, dtype=torch.uint8, device="cuda")
    grads = [torch.zeros_like(s) for s in many.shards]
    ones = torch.ones(1100, device="cuda")
    tensor = Tensor(10007, (DT.BFP16, DT.BFP16, True), True, 4)
    norm_space = torch.empty(model_ops.grad_norm_workspace(2), dtype=torch.uint8, device="cuda")
    result = torch.zeros(2, 2, device="cuda")
    count = torch.ones(1, dtype=torch.int64, device="cuda")

    def step():
        for rows, tokens, ws in ((few, few_tokens, space), (many, many_tokens, None)):
            with hccl_amd.group():
                for r, (start, n) in enumerate(rows.parts):
                    s = rows.shards[r]
                    model_ops.token_log_probs(w.comms[r], s, rows.t, start, n, tokens, rows.log_probs[r],
                                              data_type=rows.dtype, row_stride=s.stride(0), lse=rows.lse[r],
                                              entropy=rows.entropy[r], top_count=rows.top, top_values=rows.values[r],
                                              top_ids=rows.ids[r], workspace=ws, workspace_bytes=size if ws is not None else 0,
                                              stream=w.stream)
        for r, (start, n) in enumerate(many.parts):
            model_ops.token_log_probs_grad(w.comms[r], many.shards[r], 1100, start, n, many_tokens, many.lse[r], ones,
                                           grads[r], data_type=DT.FP32, row_stride=grads[r].stride(0),
                                           grad_row_stride=grads[r].stride(0), stream=w.stream)
        with hccl_amd.group():
            for r in range(2):
                model_ops.grad_norm(w.comms[r], [(tensor.view("grad"), 10007, DT.BFP16)], 0.5, result[r],
                                    workspace=norm_space, workspace_bytes=norm_space.numel(), stream=w.stream)
        model_ops.adamw(w.comms[0], [tensor.descr()], 1, 1e-3, state_type=DT.FP8E4M3, clip=result[0],
                        step_on_device=count, stream=w.stream)

    def outputs():
        return [o.clone() for rows in (few, many) for group in (rows.log_probs, rows.lse, rows.entropy, rows.values, rows.ids)
                for o in group] + [g.clone() for g in grads] + [result.clone()] + list(tensor.host().values())

    start = {k: tensor.view(k).clone() for k in tensor.rooms}

    def restart():
        for k, x in start.items():
            tensor.view(k).copy_(x)
        count.fill_(1)
        for rows in (few, many):
            for group in (rows.log_probs, rows.lse, rows.entropy, rows.values):
                for o in group:
                    o.fill_(FILL)
        result.zero_()
        torch.cuda.synchronize()

    torch.cuda.synchronize()
    eager = []
    for _ in range(3):
        step()
        w.sync()
        eager.append(outputs())
        count += 1
        few_tokens.add_(1)
        torch.cuda.synchronize()
    few_tokens.sub_(3)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=w.stream):
        step()
    restart()
    for k in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outputs(), eager[k]):
            assert torch.equal(a.float().nan_to_num(9e9), b.float().nan_to_num(9e9)), k
        count += 1
        few_tokens.add_(1)
        torch.cuda.synchronize()


def test_blocking_calls_from_one_thread_per_rank(worlds):
    """Every rank's thread, on a stream of its own, alternates these collectives with the data plane's and local steps."""
    import threading
    n, t, v = 3, 5, 3001
    w = World(n)
    try:
        x = rng_tensor(1, t, v)
        rows = Rows(x, DT.FP32, n, 4)
        tokens = given(t, v, 1)
        want = rows.run(w, tokens)
        dev = tokens.cuda()
        streams = [torch.cuda.Stream() for _ in range(n)]
        sums = [torch.zeros(100, device="cuda") for _ in range(n)]
        ones = torch.ones(100, device="cuda")
        results = torch.zeros(n, 2, device="cuda")
        spaces = [torch.empty(1 << 20, dtype=torch.uint8, device="cuda") for _ in range(n)]
        states = [[torch.zeros(100, device="cuda") for _ in range(3)] for _ in range(n)]
        errors = []
        torch.cuda.synchronize()

        def rank(r):
            try:
                start, count = rows.parts[r]
                s = rows.shards[r]
                for step in range(1, 13):
                    model_ops.token_log_probs(w.comms[r], s if count else None, t, start, count, dev, rows.log_probs[r],
                                              data_type=DT.FP32, row_stride=s.stride(0), lse=rows.lse[r],
                                              entropy=rows.entropy[r], top_count=4, top_values=rows.values[r],
                                              top_ids=rows.ids[r], workspace=spaces[r], workspace_bytes=1 << 20,
                                              stream=streams[r])
                    hccl_amd.all_reduce(w.comms[r], ones, sums[r], 100, DT.FP32, OP.SUM, streams[r])
                    model_ops.grad_norm(w.comms[r], [(sums[r], 100, DT.FP32)], 1.0, results[r], workspace=spaces[r],
                                        workspace_bytes=1 << 20, stream=streams[r])
                    model_ops.adamw(w.comms[r], [dict(param=states[r][0], grad=sums[r], exp_avg=states[r][1],
                                                      exp_avg_sq=states[r][2], count=100, param_type=DT.FP32,
                                                      grad_type=DT.FP32)], step, 0.1, clip=results[r], stream=streams[r])
            except Exception as e:      # a thread's failure must not look like success
                errors.append(e)
        threads = [threading.Thread(target=rank, args=(r,)) for r in range(n)]
        for th in threads:
            th.start()
        for th in threads:
            th.join(60)
        torch.cuda.synchronize()
        assert not errors, errors
        assert torch.equal(rows.log_probs[0][:-1].cpu().double().nan_to_num(9e9), want[0].nan_to_num(9e9))
        norm = math.sqrt(100 * n * n * n)
        assert abs(float(results[1, 0]) - norm) <= 2 * U * norm and torch.equal(results, results[:1].expand(n, 2))
        assert torch.equal(states[0][0], states[1][0]) and torch.equal(states[0][0], states[2][0])
        assert float(states[0][0].max()) < -1.0           # a dozen steps of about 0.1 against a constant gradient
    finally:
        w.close()


def test_every_replay_writes_every_output(worlds):
    """All four operators in one graph; before each replay every output, ids and gradients included, is overwritten and the
    inputs are changed.  Each replay equals the eager calls on the same inputs, made in between on other buffers."""
    if not torch.cuda.is_available():
        pytest.skip("graphs need a GPU")
    w = worlds(2)
    many_tokens, few_tokens = given(1100, 300, 2).cuda(), given(3, 50001, 1).cuda()
    weights = torch.ones(1100, device="cuda")
    count = torch.ones(1, dtype=torch.int64, device="cuda")

    class Buffers:
        def __init__(self):
            self.few = Rows(rng_tensor(1, 3, 50001), DT.BFP16, 2, 8)
            self.many = Rows(rng_tensor(2, 1100, 300), DT.FP32, 2, 4)
            self.grads = [torch.zeros_like(s) for s in self.many.shards]
            self.tensor = Tensor(10007, (DT.BFP16, DT.BFP16, True), True, 4)
            self.result = torch.zeros(2, 2, device="cuda")
            self.size = model_ops.token_log_probs_workspace(3, 50001, 8)
            self.space = torch.empty(self.size, dtype=torch.uint8, device="cuda")
            self.norm_space = torch.empty(model_ops.grad_norm_workspace(2), dtype=torch.uint8, device="cuda")

        def outputs(self):
            return [o for rows in (self.few, self.many) for kind in (rows.log_probs, rows.lse, rows.entropy, rows.values, rows.ids)
                    for o in kind] + self.grads + [self.result]

        def restart(self, k):
            """The inputs of step k; nothing left of an earlier one."""
            for o in self.outputs():
                o.fill_(77)
            for rows in (self.few, self.many):
                for s in rows.shards:
                    s.copy_((rng_tensor(40 + k, s.shape[0], s.shape[1]) * 2).to(s.dtype))
            for i, name in enumerate(sorted(self.tensor.rooms)):
                view = self.tensor.view(name)
                if view.dtype != torch.uint8:
                    view.copy_((rng_tensor(60 + 10 * k + i, *view.shape).abs() * 0.01).to(view.dtype))
                else:
                    view.fill_(40 + k)

        def step(self):
            for rows, tokens, space in ((self.few, few_tokens, self.space), (self.many, many_tokens, None)):
                with hccl_amd.group():
                    for r, (start, n) in enumerate(rows.parts):
                        s = rows.shards[r]
                        model_ops.token_log_probs(
                            w.comms[r], s, rows.t, start, n, tokens, rows.log_probs[r], data_type=rows.dtype,
                            row_stride=s.stride(0), lse=rows.lse[r], entropy=rows.entropy[r], top_count=rows.top,
                            top_values=rows.values[r], top_ids=rows.ids[r], workspace=space,
                            workspace_bytes=self.size if space is not None else 0, stream=w.stream)
            many = self.many
            for r, (start, n) in enumerate(many.parts):
                model_ops.token_log_probs_grad(
                    w.comms[r], many.shards[r], 1100, start, n, many_tokens, many.lse[r], weights, self.grads[r],
                    data_type=DT.FP32, row_stride=many.shards[r].stride(0), grad_row_stride=self.grads[r].stride(0),
                    entropy=many.entropy[r], grad_entropy=weights, top_count=4, top_ids=many.ids[r],
                    grad_top_values=many.values[r], stream=w.stream)
            with hccl_amd.group():
                for r in range(2):
                    model_ops.grad_norm(w.comms[r], [(self.tensor.view("grad"), 10007, DT.BFP16)], 0.5, self.result[r],
                                        workspace=self.norm_space, workspace_bytes=self.norm_space.numel(), stream=w.stream)
            model_ops.adamw(w.comms[0], [self.tensor.descr()], 1, 1e-3, state_type=DT.FP8E4M3, clip=self.result[0],
                            step_on_device=count, stream=w.stream)

    kept, other = Buffers(), Buffers()
    kept.restart(0)
    torch.cuda.synchronize()
    kept.step()      # (what is loaded at a first call is loaded)
    w.sync()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=w.stream):
        kept.step()
    for k in range(1, 5):
        for b in (kept, other):
            b.restart(k)
        few_tokens.add_(1)
        many_tokens[7:].copy_(torch.randint(0, 300, (1093,), generator=torch.Generator().manual_seed(k)))
        weights.copy_(rng_tensor(k, 1100))
        count.fill_(k)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        other.step()
        w.sync()
        same = lambda a, b: torch.equal(a.float().nan_to_num(9e9), b.float().nan_to_num(9e9))  # noqa: E731
        for i, (a, b) in enumerate(zip(kept.outputs(), other.outputs())):
            assert same(a, b), (k, i)
            assert bool((b != 77).any()), (k, i)
        after, want = kept.tensor.host(), other.tensor.host()
        for name in want:
            assert same(after[name], want[name]), (k, name)
        for rows in (kept.few, kept.many):      # against the definition, not only against another call
            x = torch.cat([s[:, :n].cpu() for (_, n), s in zip(rows.parts, rows.shards)], 1)
            tokens = (few_tokens if rows is kept.few else many_tokens).cpu()
            part = Rows(x, rows.dtype, 2, rows.top, parts=rows.parts)
            top = rows.top
            check_rows(part, (rows.log_probs[1][:-1].cpu().double(), rows.lse[1][:-1].cpu().double(),
                              rows.entropy[1][:-1].cpu().double(), rows.values[1][:-1].view(-1, top).cpu().double(),
                              rows.ids[1][:-1].view(-1, top).cpu().long()), tokens, 1.0)


@pytest.mark.parametrize("t,v", [(5, 3001), (3, 50001), (300, 700)])
def test_threads_that_call_for_their_ranks_leave_every_output_right(worlds, t, v):
    """A thread and a stream per rank, the inputs and every output replaced between two calls, rows shared by workgroups and
    rows that are not: all of every rank's outputs afterwards, and all threads at their end."""
    import threading
    n, top = 3, 4
    w = World(n)
    try:
        streams = [torch.cuda.Stream() for _ in range(n)]
        size = max(16, model_ops.token_log_probs_workspace(t, v, top))
        spaces = [torch.full((size,), 255, dtype=torch.uint8, device="cuda") for _ in range(n)]
        norm_space = model_ops.grad_norm_workspace(n)
        norm_spaces = [torch.full((norm_space,), 255, dtype=torch.uint8, device="cuda") for _ in range(n)]
        for seed in range(3):
            rows = Rows(rng_tensor(seed, t, v, scale=2.0), DT.FP32, n, top)
            tokens = given(t, v, seed)
            dev = tokens.cuda()
            grads = [rng_tensor(seed + r, 1000 + r) for r in range(n)]
            grads_dev = [g.cuda() for g in grads]
            results = torch.full((n, 3), FILL, device="cuda")
            errors = []
            torch.cuda.synchronize()

            def rank(r, rows=rows, dev=dev, grads_dev=grads_dev, results=results, errors=errors):
                try:
                    start, count = rows.parts[r]
                    s = rows.shards[r]
                    model_ops.token_log_probs(
                        w.comms[r], s if count else None, t, start, count, dev, rows.log_probs[r], data_type=DT.FP32,
                        row_stride=s.stride(0), lse=rows.lse[r], entropy=rows.entropy[r], top_count=top,
                        top_values=rows.values[r], top_ids=rows.ids[r], workspace=spaces[r], workspace_bytes=size,
                        stream=streams[r])
                    model_ops.grad_norm(w.comms[r], [(grads_dev[r], 1000 + r, DT.FP32)], 1.0, results[r],
                                        workspace=norm_spaces[r], workspace_bytes=norm_space, stream=streams[r])
                except Exception as e:
                    errors.append(e)
            threads = [threading.Thread(target=rank, args=(r,), daemon=True) for r in range(n)]
            for th in threads:
                th.start()
            for th in threads:
                th.join(60)
            assert not any(th.is_alive() for th in threads) and not errors, errors
            torch.cuda.synchronize()
            for r in range(n):
                got = [o[r][:-1].cpu().double() for o in (rows.log_probs, rows.lse, rows.entropy, rows.values)]
                check_rows(rows, (*got[:3], got[3].view(t, top), rows.ids[r][:-1].view(t, top).cpu().long()), tokens, 1.0)
                assert all(float(o[r][-1]) == 77 for o in (rows.log_probs, rows.lse, rows.entropy, rows.values, rows.ids))
            norm, factor = norm_reference([[(g, DT.FP32, 0)] for g in grads], 1.0, 1.0)
            for r in range(n):
                assert abs(float(results[r, 0]) - norm) <= 2 * U * norm and abs(float(results[r, 1]) - factor) <= 2 * U * factor
            assert bool((results[:, 2] == FILL).all())
    finally:
        w.close()


def test_a_sharded_training_step(worlds):
    """Two steps of a linear head, as the operators are used round the collectives: four ranks hold a quarter of the
    vocabulary's weights each and see the same rows (log probabilities and entropy over the split vocabulary, gradient of
    the part, gradients averaged over two half batches by AllReduce), then a second set of weights, replicated, whose
    gradient is reduce-scattered, clipped by the norm over everything, stepped in shards and gathered.  Against the same
    steps in 64 bits; weights of the order of one move by about lr = 0.01 per step, so that 32-bit products of 64 terms, a
    step's m / sqrt(v) being at most 1 and its relative error 1e-3 at |m| above 1e-3 of the typical, bound the distance."""
    n, t, v, width, lr = 4, 32, 1000, 64, 0.01
    w = worlds(n)
    part = v // n
    gen = torch.Generator().manual_seed(3)
    head = torch.randn(v, width, generator=gen) * 0.2
    body = torch.randn(width, width, generator=gen) * 0.2
    inputs = torch.randn(t, width, generator=gen)
    tokens = torch.randint(0, v, (t,), generator=gen)

    ref = [head.double().requires_grad_(), body.double().requires_grad_()]
    ref_state = [(torch.zeros_like(p), torch.zeros_like(p)) for p in ref]
    heads = [head[r * part:(r + 1) * part].clone().cuda() for r in range(n)]
    bodies = [body.clone().cuda() for _ in range(n)]
    share = width * width // n
    head_state = [(torch.zeros_like(h), torch.zeros_like(h)) for h in heads]
    body_state = [(torch.zeros(share, device="cuda"), torch.zeros(share, device="cuda")) for _ in range(n)]
    x, ids = inputs.cuda(), tokens.cuda()
    stream = w.stream
    for step in (1, 2):
        hidden = inputs.double() @ ref[1]
        log_p = torch.log_softmax(hidden @ ref[0].T, 1)
        loss = -log_p[torch.arange(t), tokens].mean() - 0.01 * torch.special.entr(log_p.exp()).sum(1).mean()
        grads = torch.autograd.grad(loss, ref)
        norm = math.sqrt(sum(float(g.square().sum()) for g in grads))
        factor = min(1.0, 0.5 / (norm + 1e-6))
        with torch.no_grad():
            for p, g, (m, s) in zip(ref, grads, ref_state):
                m.mul_(0.9).add_(0.1 * factor * g)
                s.mul_(0.95).add_(0.05 * (factor * g) ** 2)
                p.mul_(1 - lr * 0.1).sub_(lr / (1 - 0.9 ** step) * m / ((s / (1 - 0.95 ** step)).sqrt() + 1e-8))

        logits = [(x @ bodies[r]) @ heads[r].T for r in range(n)]
        lp, lse, ent = (torch.empty(n, t, device="cuda") for _ in range(3))
        space = torch.empty(model_ops.token_log_probs_workspace(t, v) + 16, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        with hccl_amd.group():
            for r in range(n):
                model_ops.token_log_probs(w.comms[r], logits[r], t, r * part, part, ids, lp[r], data_type=DT.FP32,
                                          lse=lse[r], entropy=ent[r], workspace=space, workspace_bytes=space.numel(),
                                          stream=stream)
        g_lp = torch.full((t,), -1.0 / t, device="cuda")
        g_ent = torch.full((t,), -0.01 / t, device="cuda")
        torch.cuda.synchronize()
        for r in range(n):
            model_ops.token_log_probs_grad(w.comms[r], logits[r], t, r * part, part, ids, lse[r], g_lp, logits[r],
                                           data_type=DT.FP32, entropy=ent[r], grad_entropy=g_ent, stream=stream)
        w.sync()
        got_loss = float(-lp[0].double().mean() - 0.01 * ent[0].double().mean())
        assert abs(got_loss - float(loss.detach())) < 1e-4
        head_grad = [logits[r].T @ (x @ bodies[r]) for r in range(n)]
        # every rank's share of the hidden state's gradient: the sum over ranks is the whole one
        body_grad = [(x.T @ (logits[r] @ heads[r])).contiguous() for r in range(n)]
        shard = [torch.empty(share, device="cuda") for _ in range(n)]
        torch.cuda.synchronize()
        with hccl_amd.group():
            for r in range(n):
                hccl_amd.reduce_scatter(w.comms[r], body_grad[r], shard[r], share, DT.FP32, OP.SUM, stream)
        result = torch.empty(n, 2, device="cuda")
        norm_space = torch.empty(model_ops.grad_norm_workspace(2 * n), dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        with hccl_amd.group():
            for r in range(n):
                model_ops.grad_norm(w.comms[r], [(head_grad[r], part * width, DT.FP32), (shard[r], share, DT.FP32)], 0.5,
                                    result[r], workspace=norm_space, workspace_bytes=norm_space.numel(), stream=stream)
        mine = [bodies[r].view(-1)[r * share:(r + 1) * share].clone() for r in range(n)]
        torch.cuda.synchronize()
        for r in range(n):
            model_ops.adamw(w.comms[r], [
                dict(param=heads[r], grad=head_grad[r], exp_avg=head_state[r][0], exp_avg_sq=head_state[r][1],
                     count=part * width, param_type=DT.FP32, grad_type=DT.FP32),
                dict(param=mine[r], grad=shard[r], exp_avg=body_state[r][0], exp_avg_sq=body_state[r][1], count=share,
                     param_type=DT.FP32, grad_type=DT.FP32)], step, lr, 0.9, 0.95, 1e-8, 0.1, clip=result[r], stream=stream)
        with hccl_amd.group():
            for r in range(n):
                hccl_amd.all_gather(w.comms[r], mine[r], bodies[r], share, DT.FP32, stream)
        w.sync()
        assert abs(float(result[0, 0]) - norm) <= 1e-4 * norm and torch.equal(result, result[:1].expand(n, 2))
        assert abs(float(result[0, 1]) - factor) <= 1e-4 * factor
        for r in range(n):
            assert torch.equal(bodies[r], bodies[0])
        # an element moves by at most about lr; where its gradient is not tiny the move itself is right to a thousandth
        for got, want, state in ((torch.cat(heads).cpu().double(), ref[0], ref_state[0]), (bodies[0].cpu().double(), ref[1], ref_state[1])):
            clear = state[0].abs() > 1e-2 * state[0].abs().mean()
            off = (got - want.detach()).abs()
            assert float(off[clear].max()) < 2e-2 * lr and float(off.max()) < 2.5 * step * lr
