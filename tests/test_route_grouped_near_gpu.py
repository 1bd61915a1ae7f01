"""route_grouped_topk where choices lie close together, against the order of
64-bit values: groups that tie exactly, a few near experts among far ones, sums
of a group that differ by less than f32 holds, scores that f32 cannot hold."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64
SCORINGS = ["softmax", "sigmoid", "sqrtsoftplus"]


@pytest.fixture(scope="module")
def dw():
    import dw_tpu_b200
    return dw_tpu_b200


@pytest.fixture(autouse=True)
def _no_device_error():
    yield
    from dw_tpu_b200 import _lib
    _lib.raise_on_device_error()


def _scores(x, scoring):
    if scoring == "softmax":
        return torch.softmax(x, 1)
    if scoring == "sigmoid":
        return 1 / (1 + torch.exp(-x))
    return (x.clamp(min=0) + torch.log1p(torch.exp(-x.abs()))).sqrt()


def _ref(x, k, groups, keep, renorm, scoring, group_score, scale, bias):
    """(weights, ids, undecided rows) in 64 bits: values descending, ties to the
    lower index, without a bias by the logits. Undecided: groups of unlike pairs of
    experts on both sides of the border, whose sums lie within 2^-44 of the row's
    largest |score| + |bias|, or (with a bias) two unlike experts in a row that do. A
    score is off by a few steps of 2^-53 of itself, under softmax by those of a sum of
    1024 (some 2^-47), here and in the kernel; the difference of two sums of two such
    values, twice, by less than 2^-44."""
    x = x.double().cpu()
    t, e = x.shape
    per = e // groups
    s = _scores(x, scoring)
    b = torch.zeros(e, dtype=F64) if bias is None else bias.double().cpu()
    c = x if bias is None else s + b
    cg = c.reshape(t, groups, per)
    at = cg.sort(dim=2, descending=True, stable=True)[1][:, :, :1 if group_score == "max" else 2]
    pairs = x.reshape(t, groups, per).gather(2, at)
    if group_score == "max":
        v = cg.amax(2)
    else:
        v = (s + b if bias is not None else s).reshape(t, groups, per).gather(2, at).sum(2)
    by = v.sort(dim=1, descending=True, stable=True)[1]
    undecided = torch.zeros(t, dtype=torch.bool)
    slack = 2.0 ** -44 * (s + b.abs()).amax(1, keepdim=True)
    if keep < groups and group_score == "top2":
        in_order = v.gather(1, by)
        near = (v - in_order[:, keep - 1:keep]).abs() <= slack
        like = torch.cat([pairs, b.expand(t, e).reshape(t, groups, per).gather(2, at)], 2)
        most = torch.where(near[:, :, None], like, -math.inf).amax(1)
        least = torch.where(near[:, :, None], like, math.inf).amin(1)
        outside = in_order[:, keep - 1] - in_order[:, keep] <= slack[:, 0]
        undecided = outside & ~(most == least).all(1)
    open_ = torch.zeros((t, groups), dtype=torch.bool).scatter_(1, by[:, :keep], True)
    order = c.sort(dim=1, descending=True, stable=True)[1]
    is_open = open_.repeat_interleave(per, 1).gather(1, order)
    ids = order.gather(1, (~is_open).to(torch.int8).sort(dim=1, stable=True)[1])[:, :k + 1]
    if bias is not None and k < keep * per:
        picked, logit, of = c.gather(1, ids), x.gather(1, ids), b[ids]
        unlike = (logit[:, 1:] != logit[:, :-1]) | (of[:, 1:] != of[:, :-1])
        undecided |= ((picked[:, :-1] - picked[:, 1:] <= slack) & unlike).any(1)
    ids = ids[:, :k]
    w = s.gather(1, ids)
    if renorm:
        total = w.sum(1, keepdim=True)
        w = torch.where(total == 0, torch.zeros_like(w), w / total)
    return w * scale, ids.int(), undecided


def _check(dw, x, k, groups, keep, scoring="sigmoid", group_score="top2", bias=None, renorm=True,
           scale=2.5):
    w, ids = dw.route_grouped_topk(x, k, groups, keep, renorm, scoring, group_score, scale, F32,
                                   bias)
    rw, ri, undecided = _ref(x, k, groups, keep, renorm, scoring, group_score, scale, bias)
    assert int(undecided.sum()) <= len(x) // 20
    sure = ~undecided
    wrong = (ids.cpu() != ri).any(1) & sure
    assert not wrong.any(), (
        f"{int(wrong.sum())} of {len(x)} tokens, first {int(wrong.nonzero()[0])}: "
        f"{ids[wrong.nonzero()[0]].tolist()} for {ri[wrong.nonzero()[0]].tolist()}")
    # Steps of f32 (2^-24) of a weight: 4 of expf, 1 each of 1 + e, the division, the
    # renormalisation and the scale; of a total of at most 32 such weights as many and 8
    # more; of a softmax's sum 4 of expf, the mean size of its exponents (ln 256 at
    # most) and some 10 additions. Below 2^5.
    err = (w.cpu().double() - rw).abs()[sure]
    assert bool((err <= 2.0 ** -19 * rw[sure].abs() + 1e-37).all()), float(err.max())
    return w, ids


def _steps(value, n):
    """The f32 numbers 0, 1, .. n - 1 steps above ``value``."""
    return (torch.tensor(value).view(torch.int32) + torch.arange(n, dtype=torch.int32)).view(F32)


@pytest.mark.parametrize("e,groups", [(112, 4), (84, 3), (104, 2), (112, 2), (120, 2), (240, 2),
                                      (56, 2), (28, 1)])
@pytest.mark.parametrize("scoring", SCORINGS)
def test_groups_that_tie_where_lanes_are_left_over(dw, e, groups, scoring):
    """Groups that the lanes of a warp do not share out evenly, logits of four values:
    most tokens have two groups of one value."""
    g = torch.Generator().manual_seed(e + groups)
    level = torch.tensor([0.0, 0.0, 0.0, 0.5, 0.75, 1.0])
    for t in (1, 200):
        x = level[torch.randint(0, 6, (t, e), generator=g)] * (torch.rand((t, e), generator=g) < 0.2)
        x = x.cuda()
        for bias in (None, torch.full((e,), 0.25, device="cuda"),
                     (torch.randint(0, 2, (e,), generator=g) * 0.5).cuda()):
            for gs in ("max", "top2"):
                if gs == "top2" and bias is not None and bias.unique().numel() > 1:
                    continue  # (sums of unlike scores and biases tie by rounding)
                for keep in range(1, groups + 1):
                    for k in (1, 4):
                        _check(dw, x, k, groups, keep, scoring, gs, bias)


def test_empty_lanes_add_no_expert_to_a_group(dw):
    x = torch.zeros((1, 112))
    x[0, 0], x[0, 1] = 1.0, 0.5
    x[0, 28] = x[0, 56] = 1.0
    x[0, 29] = x[0, 57] = 0.75
    _, ids = _check(dw, x.cuda(), 1, 4, 1)
    assert ids.item() == 28


@pytest.mark.parametrize("steps", [(2, 1, 3), (1, 1, 2), (3, 1, 5), (0, 0, 1, 4), (4, 0, 2, 7)])
@pytest.mark.parametrize("e,groups", [(32, 1), (256, 8), (512, 1), (1024, 4)])
def test_experts_of_one_lane_steps_apart(dw, steps, e, groups):
    """The experts left after the last pick decide too, not the first of them alone."""
    near = _steps(1.0, 8)
    for at in (0, 5, e // groups - 4):
        x = torch.full((1, e), 0.5)
        for j, s in enumerate(steps):
            x[0, at + j] = near[s]
        for t in (1, 2001):
            y = x.expand(t, e).cuda()
            for k in (1, 2, 3):
                for scoring in SCORINGS:
                    _check(dw, y.contiguous(), k, groups, groups, scoring, "max")
    zero = torch.zeros(e, device="cuda")
    x = torch.full((1, e), -1.0, dtype=BF)
    x[0, :3] = torch.tensor([11.0, 11.0, 11.0625])  # sigmoids 1.0e-6 apart
    for k in (1, 2, 3):
        _check(dw, x.cuda(), k, groups, groups, bias=zero)


def _near_among_far(seed, t, e, top_k, run=None):
    """Tokens of far logits with 2 to 4 within 7 steps of 1 across the cut at top_k, within
    ``run`` neighbours or anywhere, and the larger ones well above."""
    g = torch.Generator().manual_seed(seed)
    x = -2 * torch.rand((t, e), generator=g)
    near = _steps(1.0, 8)
    for i in range(t):
        n = int(torch.randint(2, 5, (1,), generator=g))
        below = int(torch.randint(1, min(top_k, n - 1) + 1, (1,), generator=g))
        places = torch.randperm(e, generator=g)
        if run:
            first = int(torch.randint(0, e // run, (1,), generator=g)) * run
            inside = first + torch.randperm(run, generator=g)[:n]
            rest = places[(places < first) | (places >= first + run)]
            places = torch.cat([inside, rest])
        x[i, places[:n]] = near[torch.randint(0, 8, (n,), generator=g)]
        larger = top_k - below
        x[i, places[n:n + larger]] = 2 + torch.randperm(32, generator=g)[:larger] / 8
    return x


@pytest.mark.parametrize("top_k", [1, 2, 8])
@pytest.mark.parametrize("t", [1, 200, 2001])
@pytest.mark.parametrize("e,groups,run", [(256, 8, 8), (256, 8, None), (128, 1, 16), (160, 8, 20),
                                          (64, 4, None)])
def test_near_experts_among_far_ones(dw, top_k, t, e, groups, run):
    x = _near_among_far(top_k + t + e, max(t, 60), e, top_k, run)
    flat = torch.full((e,), 0.25)
    one = torch.zeros(e)
    one[::3] = 2.0 ** -20
    tokens = [x.cuda()] if t > 1 else [row[None].cuda() for row in x]
    for y in tokens:
        for scoring in SCORINGS:
            for gs in ("max", "top2"):
                _check(dw, y, top_k, groups, groups, scoring, gs)
                _check(dw, y, top_k, groups, groups, scoring, gs, flat.cuda())
        _check(dw, y, top_k, groups, groups, bias=one.cuda())


@pytest.mark.parametrize("e,groups,keep", [(256, 8, 8), (256, 8, 4), (160, 8, 3), (256, 1, 1)])
@pytest.mark.parametrize("offset", [50.0, -50.0, 1000.0])
def test_a_common_offset_of_the_logits(dw, e, groups, keep, offset):
    """Softmax scores are those without the offset; the logits' steps are 4e-6 to 6e-5."""
    g = torch.Generator().manual_seed(int(offset) + e)
    x = (torch.randn((1500, e), generator=g) * 1e-3 + offset).cuda()
    spread = (torch.randn((1500, e), generator=g) * 1.5 + offset).cuda()
    b = (torch.randn(e, generator=g) * 0.01).cuda()
    for y in (x, spread):
        for k in (1, 2, 4, 8):
            _check(dw, y, k, groups, keep, "softmax", "max")
        _check(dw, y, 8, groups, keep, "softmax", "top2")
        _check(dw, y, 8, groups, keep, "softmax", "top2", b, scale=1.0)


def _near_groups(seed, t, e, groups):
    """Groups whose largest lie 0 to 6 steps apart, each with a second one as near."""
    g = torch.Generator().manual_seed(seed)
    per = e // groups
    x = -1 - torch.rand((t, groups, per), generator=g)
    near = _steps(1.0, 7)
    for i in range(t):
        for q in range(groups):
            if torch.rand((), generator=g) < 0.6:
                n = min(per, int(torch.randint(1, 4, (1,), generator=g)))
                first = int(torch.randint(0, per - n + 1, (1,), generator=g))
                x[i, q, first:first + n] = near[torch.randint(0, 7, (n,), generator=g)]
    return x.reshape(t, e)


@pytest.mark.parametrize("e,groups,keep,k", [(160, 8, 1, 1), (256, 8, 4, 8), (256, 8, 1, 2),
                                             (64, 16, 5, 4), (1024, 4, 2, 8), (96, 3, 1, 1)])
@pytest.mark.parametrize("t", [100, 2001])
def test_groups_whose_best_are_steps_apart(dw, e, groups, keep, k, t):
    x = _near_groups(e + keep, t, e, groups).cuda()
    b = torch.full((e,), 0.25, device="cuda")
    for scoring in SCORINGS:
        _check(dw, x, k, groups, keep, scoring, "max")
        _check(dw, x, k, groups, keep, scoring, "max", b)


@pytest.mark.parametrize("top_k", [1, 2, 8])
@pytest.mark.parametrize("e,groups", [(256, 8), (160, 8), (96, 3)])
def test_near_experts_with_a_group_closed(dw, top_k, e, groups):
    x = _near_among_far(top_k + e, 2001, e, top_k).cuda()
    for scoring in SCORINGS:
        for keep in (groups - 1, max(1, groups // 2)):
            _check(dw, x, top_k, groups, keep, scoring, "max")
            _check(dw, x[:200], top_k, groups, keep, scoring, "max")


def test_the_largest_of_a_group_and_not_its_first(dw):
    near = _steps(1.0, 8)
    for t in (1, 2001):
        x = torch.full((t, 160), 0.5)
        x[:, 0], x[:, 1], x[:, 20] = near[0], near[5], near[3]
        _, ids = _check(dw, x.cuda(), 1, 8, 1, group_score="max")
        assert bool((ids == 1).all())


@pytest.mark.parametrize("e,groups,keep", [(256, 8, 4), (160, 8, 3), (1024, 1, 1)])
@pytest.mark.parametrize("low", [-12.0, -30.0, -60.0, -95.0])
def test_biases_as_small_as_the_scores(dw, e, groups, keep, low):
    """Strongly negative logits: the scores are e^low, and so are the biases, so that the
    error of the exponential counts whole."""
    g = torch.Generator().manual_seed(int(-low) + e)
    x = (low + torch.rand((4000, e), generator=g) * 0.5).cuda()
    for scoring in ("sigmoid", "sqrtsoftplus"):
        size = math.exp(low if scoring == "sigmoid" else low / 2)
        b = (torch.rand(e, generator=g, dtype=F64) * size).to(F32).cuda()
        for gs in ("max", "top2"):
            _check(dw, x, 8, groups, keep, scoring, gs, b)


def _two_choices(seed, t, e, low, scoring):
    """(logits, biases): two experts of each token whose choices differ by less than a step
    of the larger logit, by way of biases a thousandth of the scores; the others far below."""
    g = torch.Generator().manual_seed(seed)
    score = (lambda v: 1 / (1 + torch.exp(-v))) if scoring == "sigmoid" else (
        lambda v: torch.log1p(torch.exp(v)).sqrt())
    per = 1 if scoring == "sigmoid" else 2  # log score is about the logit / per
    b = (torch.rand(e, generator=g, dtype=F64) * float(score(torch.tensor(low, dtype=F64))) *
         1e-3).to(F32)
    x = torch.full((t, e), low - 3, dtype=F32)
    i, j = torch.rand((t, e), generator=g).topk(2, dim=1)[1].unbind(1)
    rows = torch.arange(t)
    x[rows, i] = low + torch.rand(t, generator=g) * 0.01
    want = score(x[rows, i].double()) + b[i].double() - b[j].double()
    v = x[rows, i].double()
    for _ in range(8):
        v = v + per * torch.log(want / score(v))
    x[rows, j] = v.to(F32)
    return x, b


@pytest.mark.parametrize("low", [-6.0, -20.0, -40.0, -60.0, -80.0])
@pytest.mark.parametrize("scoring", ["sigmoid", "sqrtsoftplus"])
def test_two_near_choices_of_tiny_scores(dw, scoring, low):
    x, b = _two_choices(int(-low), 4000, 256, low, scoring)
    for groups, keep in ((1, 1), (8, 8), (8, 1)):
        _check(dw, x.cuda(), 1, groups, keep, scoring, "max", b.cuda())
        _check(dw, x[:500].cuda(), 1, groups, keep, scoring, "max", b.cuda())


def test_many_experts_under_a_biased_softmax(dw):
    """The sum over all the experts is in every choice."""
    g = torch.Generator().manual_seed(5)
    for e, groups, keep in ((1024, 1, 1), (1024, 8, 4), (256, 8, 4)):
        x = (torch.randn((4000, e), generator=g) * 2).cuda()
        b = (torch.randn(e, generator=g) / e).cuda()
        for gs in ("max", "top2"):
            _check(dw, x, 8, groups, keep, "softmax", gs, b)


@pytest.mark.parametrize("scoring", SCORINGS)
@pytest.mark.parametrize("low", [-82.0, -89.0, -95.0, -105.0, -200.0])
@pytest.mark.parametrize("t", [1, 300])
def test_weights_of_scores_below_f32(dw, scoring, low, t):
    """Scores that f32 does not hold still have ratios; a few ordinary tokens among them,
    masked ones, and chosen experts far below a closed group's."""
    g = torch.Generator().manual_seed(int(-low))
    x = low + torch.rand((t, 64), generator=g) * 4
    if t > 1:
        x[::7] = torch.randn((len(x[::7]), 64), generator=g)
        x[3, 5:] = -math.inf
        x[10, 3:] = -3.0e38
    for renorm in (True, False):
        for groups, keep in ((1, 1), (8, 3)):
            _check(dw, x.cuda(), 8, groups, keep, scoring, renorm=renorm)
    if scoring != "softmax":
        return
    b = torch.zeros(64)
    b[32:] = 10 + torch.arange(32) / 8
    x = low + torch.rand((t, 64), generator=g) * 4
    x[:, :32] += -low
    for renorm in (True, False):
        _check(dw, x.cuda(), 8, 8, 3, scoring, bias=b.cuda(), renorm=renorm)


@pytest.mark.parametrize("e,groups,keep,k", [(1, 1, 1, 1), (64, 8, 3, 4), (250, 5, 2, 8),
                                             (1024, 32, 1, 32), (33, 1, 1, 32)])
@pytest.mark.parametrize("t", [0, 1, 5, 1500])
def test_logits_of_64_bits(dw, e, groups, keep, k, t):
    """Logits that f32 rounds to one number keep their order."""
    g = torch.Generator().manual_seed(e + t)
    x = torch.randn((t, e), generator=g, dtype=F64).cuda()
    close = 1 + torch.randperm(t * e, generator=g).reshape(t, e).to(F64) * 2.0 ** -45
    b = (torch.randint(0, 3, (e,), generator=g) * 0.25).cuda()
    for scoring in SCORINGS:
        for gs in ("max", "top2"):
            _check(dw, x, k, groups, keep, scoring, gs)
            _check(dw, x, k, groups, keep, scoring, gs, b, renorm=False)
        _check(dw, close.cuda(), k, groups, keep, scoring, "max")


def test_64_bit_logits_padding_strides_and_types(dw):
    g = torch.Generator().manual_seed(3)
    wide = torch.full((9, 70), math.nan, dtype=F64)
    wide[:, 3:67] = torch.randn((9, 64), generator=g, dtype=F64)
    x = wide.cuda()[:, 3:67]
    w, ids = dw.route_grouped_topk(x, 4, 8, 2, dtype=F32, num_valid_tokens=7)
    rw, ri, _ = _ref(x, 4, 8, 2, True, "sigmoid", "top2", 1.0, None)
    rw[7:], ri[7:] = 0, 0
    assert torch.equal(ids.cpu(), ri)
    assert bool(((w.cpu().double() - rw).abs() <= 2.0 ** -24 * rw).all())  # one rounding
    y = x.clone()
    y[2, 5], y[3] = math.nan, -math.inf
    w2, ids2 = dw.route_grouped_topk(y, 4, 8, 2, dtype=F32, num_valid_tokens=7)
    rest = [0, 1, 4, 5, 6]
    assert torch.equal(w2[rest], w[rest]) and torch.equal(ids2[rest], ids[rest])
    assert 5 not in ids2[2].tolist() and not bool(w2[3].any())
    # Whole numbers past 2^24, and half precision, as they are.
    n = (2 ** 24 + torch.randperm(64, generator=g))[None].cuda()
    assert dw.route_grouped_topk(n, 4, 1, 1, group_score="max")[1].tolist() == \
        n.argsort(1, descending=True)[:, :4].tolist()
    h = torch.randn((20, 64), generator=g).half().cuda()
    _check(dw, h, 4, 8, 2)


@pytest.mark.parametrize("per", list(range(1, 41)) + [63, 64, 100, 128])
def test_groups_of_every_size(dw, per):
    """Every length of a lane's run, by itself in a lane or over several."""
    g = torch.Generator().manual_seed(per)
    for t in (9, 2001):
        x = torch.randn((t, 8 * per), generator=g) * 1.5
        x[::3] = _near_groups(per, len(x[::3]), 8 * per, 8)
        b = (torch.randn(8 * per, generator=g) * 0.1).cuda()
        for dtype in (F32, BF):
            y = x.to(dtype).cuda()
            _check(dw, y, min(6, 3 * per), 8, 3, "softmax", "max")
            _check(dw, y, min(6, 3 * per), 8, 3, "sigmoid", "top2", b)
