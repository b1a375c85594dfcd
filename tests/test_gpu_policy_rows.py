"""Priors, log-probabilities, the policy loss and the preference loss on the GPU against the 64-bit oracle
(tests/learn_oracle.py, where the tolerances are derived), through the public entry points."""
import math

import numpy as np
import pytest

from tests import learn_oracle as O

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def learner():
    import omoknuni_small_amd as omk
    return omk.Learner()


def near(got, want, off, what):
    got = got.detach().double().cpu().numpy() if hasattr(got, "detach") else got
    assert got.shape == np.shape(want), what
    assert (np.isnan(got) == np.isnan(want)).all(), what
    with np.errstate(invalid="ignore"):
        wrong = ~((np.abs(got - want) <= off) | (got == want) | np.isnan(want))
    if wrong.any():
        at = np.argwhere(wrong)[0]
        raise AssertionError("%s: %d of %d, first at %s: %r for %r, %.3g off, %.3g allowed" % (
            what, wrong.sum(), wrong.size, at.tolist(), got[tuple(at)], np.asarray(want)[tuple(at)],
            abs(got[tuple(at)] - np.asarray(want)[tuple(at)]), np.broadcast_to(off, wrong.shape)[tuple(at)]))


class Case:
    """Rows with everything that a row can have: no legal action, one, -inf and lowest logits among the legal, NaN and
    infinities among the illegal, moves outside the action space and illegal moves."""

    def __init__(self, seed, rows, actions, kind, legal=None, spread=3.0, stride=0, shared=False, odd=True):
        rng = np.random.default_rng(seed)
        dtype = TYPES[kind]
        self.kind, self.rows, self.actions = kind, rows, actions
        x = rng.normal(0, spread, (rows, actions))
        mask = None
        if legal is not None:
            mask = rng.random((1 if shared else rows, actions)) < legal
            mask[np.arange(len(mask)), rng.integers(0, actions, len(mask))] = True
            if odd and not shared and rows >= 8:
                mask[3] = False
                mask[5] = False
                mask[5, actions - 1] = True
            mask = np.broadcast_to(mask, (rows, actions))
        if odd and rows >= 8:
            x[1, rng.integers(0, actions, actions // 3 + 1)] = -np.inf
            x[2] = float(torch.finfo(dtype).min)
            x[6] = -np.inf
            x[7, 0] = float(torch.finfo(dtype).min)
        # what stands in illegal columns is never looked at
        dirty = x.copy()
        if mask is not None:
            junk = rng.choice([np.nan, np.inf, -np.inf, 1e30], (rows, actions))
            dirty = np.where(mask, x, junk)
        wide = torch.full((rows, actions + stride), float("nan"), dtype=dtype)
        wide[:, :actions] = torch.from_numpy(dirty).to(dtype)
        self.wide = wide.cuda()
        self.logits = self.wide[:, :actions]
        held = torch.from_numpy(x).to(dtype).double().numpy()
        self.oracle = O.Rows(held, mask)
        self.legal = None
        if mask is not None:
            import omoknuni_small_amd as omk
            packed = omk.pack_legal(torch.from_numpy(mask[:1].copy() if shared else mask.copy()))
            self.legal = (packed[0] if shared else packed).cuda()
        moves = self.oracle.p.cumsum(1) > rng.random((rows, 1))
        self.moves = moves.argmax(1).astype(np.int32)
        if odd and rows >= 8:
            self.moves[0] = -1
            self.moves[4] = actions
        self.d_moves = torch.from_numpy(self.moves).cuda()
        self.rng = rng


SIZES = [(1, 1), (1, 2), (3, 31), (9, 32), (64, 33), (257, 63), (8, 64), (8, 65), (33, 218), (70, 225), (41, 362), (9, 1000),
         (12, 2049), (8, 4097), (9, 8192), (8, 20011), (3, 70001)]


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,actions", SIZES)
@pytest.mark.parametrize("legal", [None, 0.5])
def test_priors_and_logprobs(learner, rows, actions, kind, legal):
    c = Case(rows * 7 + actions, rows, actions, kind, legal)
    o = c.oracle
    near(learner.priors(c.logits, legal=c.legal), o.p, o.priors_off(), "priors")
    got = learner.logprobs(c.logits, c.d_moves, legal=c.legal, entropy=True)
    lp, counts, off = o.taken(c.moves)
    inside = (c.moves >= 0) & (c.moves < actions)
    lp = np.where(inside & ~counts, -np.inf, lp)
    near(got.logprob, lp, np.where(counts, off + np.abs(lp) * O.U, 0.0), "logprob")
    near(got.entropy, o.entropy, o.entropy_off(), "entropy")
    assert learner.logprobs(c.logits, legal=c.legal, entropy=True).logprob is None


def columns(c, spread=0.3):
    lp, counts, _ = c.oracle.taken(c.moves)
    old = (lp + c.rng.normal(0, spread, c.rows)).astype(np.float32)
    ref = (lp + c.rng.normal(0, 2 * spread, c.rows)).astype(np.float32)
    adv = c.rng.normal(0, 1, c.rows).astype(np.float32)
    weight = c.rng.uniform(0.5, 1.5, c.rows).astype(np.float32)
    if c.rows >= 16:
        adv[8] = 0.0
        weight[9] = 0.0
        ref[10] = np.float32(lp[10])  # nothing to pay
        old[11] = np.float32(lp[11])
    # rows that are left out: whatever their columns hold
    for column in (old, ref, adv, weight):
        column[~counts] = np.nan
    return old, adv, ref, weight


def policy_case(learner, c, clip_low=0.2, clip_high=0.28, kl_weight=0.05, use_ref=True, use_weight=True, grad=True):
    old, adv, ref, weight = columns(c)
    want = O.policy_loss(c.oracle, c.moves, old.astype(np.float64), adv.astype(np.float64),
                         ref.astype(np.float64) if use_ref else None, weight.astype(np.float64) if use_weight else None,
                         clip_low, clip_high, kl_weight if use_ref else 0.0, 1.0 / c.rows)
    d = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    got = learner.policy_loss(c.logits, c.d_moves, d(old), d(adv), ref_logprob=d(ref) if use_ref else None,
                              weight=d(weight) if use_weight else None, legal=c.legal, clip_low=clip_low,
                              clip_high=clip_high, kl_weight=kl_weight if use_ref else 0.0, grad=grad)
    for name in ("logprob", "kl", "loss"):
        near(getattr(got, name), *want[name], name)
    if grad is not False:
        near(got.grad, *c.oracle.gradient(c.moves, *want["slope"], c.kind), "grad")
    return got


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,actions", SIZES)
@pytest.mark.parametrize("legal", [None, 0.5])
def test_policy_loss(learner, rows, actions, kind, legal):
    c = Case(rows * 11 + actions, rows, actions, kind, legal)
    policy_case(learner, c, use_ref=actions % 2 == 1, use_weight=rows % 2 == 1)


@pytest.mark.parametrize("kind,actions", [("f32", 4), ("f32", 33), ("f32", 101), ("f32", 225), ("f32", 256), ("f32", 499),
                                          ("bf16", 7), ("bf16", 8), ("bf16", 9), ("bf16", 225), ("f16", 362), ("bf16", 504), ("f16", 999)])
@pytest.mark.parametrize("layout", ["together", "apart", "in place", "shifted"])
def test_many_narrow_rows(learner, kind, actions, layout):
    """As many rows as are taken several to a wavefront, where the end of one and the beginning of the next share 16 bytes:
    rows that follow one another, rows with a gap, gradients in the logits' place and ones whose vectors lie
    elsewhere."""
    rows = 8192 + 37
    c = Case(actions, rows, actions, kind, 0.5 if layout != "apart" else None, stride=3 if layout == "apart" else 0)
    near(learner.priors(c.logits, legal=c.legal), c.oracle.p, c.oracle.priors_off(), "priors")
    got = learner.logprobs(c.logits, c.d_moves, legal=c.legal, entropy=True)
    near(got.entropy, c.oracle.entropy, c.oracle.entropy_off(), "entropy")
    grad = True
    if layout == "in place":
        grad = c.logits
    elif layout == "shifted":
        out = torch.full((rows * actions + 9,), 9.0, dtype=TYPES[kind], device="cuda")
        grad = out[1:1 + rows * actions].view(rows, actions)
    policy_case(learner, c, grad=grad)
    if layout == "shifted":
        assert out[0] == 9 and (out[1 + rows * actions:] == 9).all()


@pytest.mark.parametrize("clip_low,clip_high,kl_weight", [(0.0, 0.0, 0.0), (1.0, 4.0, 1.0), (2.5, 0.1, 0.0)])
def test_policy_loss_borders(learner, clip_low, clip_high, kl_weight):
    policy_case(learner, Case(5, 200, 225, "f32", 0.4), clip_low, clip_high, kl_weight)


@pytest.mark.parametrize("actions", [225, 362, 5000, 40000])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_strides_in_place_and_shared_masks(learner, actions, kind):
    for stride in (1, 7, 64):
        c = Case(stride, 37, actions, kind, 0.5, stride=stride, shared=True)
        policy_case(learner, c)
        c = Case(stride, 37, actions, kind, 0.5, stride=stride)
        behind = c.wide[:, actions:].clone()
        got = policy_case(learner, c, grad=c.logits)
        assert got.grad.data_ptr() == c.logits.data_ptr()
        assert torch.equal(behind.isnan(), c.wide[:, actions:].isnan())
    # a gradient with another stride than the logits', and rows that begin at any address of their type
    c = Case(3, 37, actions, kind, None)
    flat = torch.zeros(37 * actions + 5, dtype=TYPES[kind], device="cuda")
    shifted = flat[5:].view(37, actions)
    shifted.copy_(c.logits)
    c.logits = shifted
    out = torch.full((37, actions + 3), 9.0, dtype=TYPES[kind], device="cuda")
    policy_case(learner, c, grad=out[:, 1:actions + 1])
    assert (out[:, 0] == 9).all() and (out[:, actions + 1:] == 9).all()
    priors = torch.full((37, actions + 3), 9.0, device="cuda")
    near(learner.priors(c.logits, out=priors[:, 2:actions + 2]), c.oracle.p, c.oracle.priors_off(), "priors")
    assert (priors[:, :2] == 9).all() and (priors[:, actions + 2:] == 9).all()


@pytest.mark.parametrize("actions", [5, 300, 3000, 50000])
def test_numbers_that_are_none(learner, actions):
    """A NaN or +inf among a row's legal logits shows in that row and in no other; one row without a number in its columns
    likewise."""
    x = torch.randn(6, actions, device="cuda")
    x[1, actions // 2] = math.nan
    x[4, 1] = math.inf
    moves = torch.zeros(6, dtype=torch.int32, device="cuda")
    ones = torch.ones(6, device="cuda")
    lp = learner.logprobs(x, moves, entropy=True)
    bad = torch.tensor([False, True, False, False, True, False], device="cuda")
    assert torch.equal(lp.logprob.isnan(), bad) and torch.equal(lp.entropy.isnan(), bad)
    assert torch.equal(learner.priors(x).isnan().any(1), bad)
    got = learner.policy_loss(x, moves, lp.logprob.nan_to_num(), ones)
    assert torch.equal(got.grad.isnan().any(1), bad) and got.loss.isnan()
    ones[2] = math.nan
    x = torch.randn(6, actions, device="cuda")
    got = learner.policy_loss(x, moves, learner.logprobs(x, moves).logprob, ones)
    assert got.grad.isnan().any(1).tolist() == [False, False, True, False, False, False]


@pytest.mark.parametrize("actions", [300, 3000, 70000])
def test_rows_of_weight_0_and_a_divergence_that_is_only_reported(learner, actions):
    x = torch.randn(9, actions, device="cuda")
    moves = torch.arange(9, dtype=torch.int32, device="cuda")
    lp = learner.logprobs(x, moves).logprob
    adv, weight, ref = torch.ones(9, device="cuda"), torch.ones(9, device="cuda"), lp.clone()
    old = lp.clone()
    weight[4], old[4], adv[5], weight[5], ref[6], weight[6] = 0, math.nan, math.inf, 0, math.inf, 0
    got = learner.policy_loss(x, moves, old, adv, ref_logprob=ref, weight=weight, kl_weight=0.5)
    rest = [0, 1, 2, 3, 7, 8]
    want = learner.policy_loss(x[rest], moves[rest], lp[rest], adv[rest], ref_logprob=lp[rest], kl_weight=0.5, scale=1 / 9)
    assert (got.grad[4:7] == 0).all() and torch.equal(got.grad[rest], want.grad)
    assert abs(float(got.loss - want.loss)) <= 4 * O.U
    # a reference that gives a move all but no chance: its divergence passes the largest float, and is weighed with 0
    ref = lp + 100.0
    got = learner.policy_loss(x, moves, lp, torch.ones(9, device="cuda"), ref_logprob=ref)
    assert got.kl.isinf().all() and got.loss.isfinite() and got.grad.isfinite().all()


def preference_case(learner, c, lengths, beta=0.3, smoothing=0.1, before=0, use_ref=True, grad=True):
    begin = before + np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
    lp, counts, _ = c.oracle.taken(c.moves)
    ref = None
    if use_ref:
        sums = np.array([lp[a:b].sum() for a, b in zip(begin, begin[1:])])
        ref = (sums + c.rng.normal(0, 2, len(sums))).astype(np.float32)
    pairs = len(lengths) // 2
    want = O.preference_loss(c.oracle, c.moves, begin, None if ref is None else ref.astype(np.float64), beta, smoothing, 1.0 / pairs)
    got = learner.preference_loss(c.logits, c.d_moves, torch.from_numpy(begin).cuda(),
                                  ref_logprob=None if ref is None else torch.from_numpy(ref).cuda(), legal=c.legal,
                                  beta=beta, label_smoothing=smoothing, grad=grad)
    for name in ("logprob", "margin", "loss"):
        near(getattr(got, name), *want[name], name)
    if grad is not False:
        g, off = c.oracle.gradient(c.moves, *want["slope"], c.kind)
        first, last = int(begin[0]), int(begin[-1])
        near(got.grad[first:last], g[first:last], off[first:last], "grad")
        if grad is True:
            assert (got.grad[:first] == 0).all() and (got.grad[last:] == 0).all()
    return got


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("actions", [1, 2, 33, 225, 362, 1000, 4097, 20011])
@pytest.mark.parametrize("lengths", [(1, 1), (5, 0), (0, 0, 3, 9), (40, 17, 1, 90, 0, 64), tuple(range(1, 15))], ids=str)
def test_preference_loss(learner, kind, actions, lengths):
    for legal, before, behind in ((None, 0, 0), (0.5, 3, 2)):
        c = Case(actions + len(lengths), before + sum(lengths) + behind, actions, kind, legal)
        preference_case(learner, c, lengths, before=before, use_ref=legal is None,
                        smoothing=0.0 if actions == 225 else 0.1)


def test_preference_leaves_other_rows(learner):
    c = Case(1, 60, 362, "bf16", 0.5)
    out = torch.full_like(c.logits, 7.0)
    preference_case(learner, c, (10, 20, 5, 5), before=9, grad=out)
    assert (out[:9] == 7).all() and (out[49:] == 7).all()
    preference_case(learner, c, (10, 20, 5, 5), before=9, grad=False)
    preference_case(learner, c, (10, 20, 5, 5), before=9, grad=c.logits)  # in place, the last use of these logits


def test_line_bounds_outside_the_rows(learner):
    """Bounds that do not fit are taken as the nearest that do, and a line that ends before it begins is empty."""
    c = Case(2, 50, 225, "f32", None)
    got = learner.preference_loss(c.logits, c.d_moves, torch.tensor([-5, 20, 900], dtype=torch.int32, device="cuda"))
    want = learner.preference_loss(c.logits, c.d_moves, torch.tensor([0, 20, 50], dtype=torch.int32, device="cuda"))
    assert torch.equal(got.logprob, want.logprob) and torch.equal(got.grad, want.grad) and torch.equal(got.loss, want.loss)
    got = learner.preference_loss(c.logits, c.d_moves, torch.tensor([40, 20, 2 ** 31 - 1], dtype=torch.int32, device="cuda"))
    want = learner.preference_loss(c.logits, c.d_moves, torch.tensor([40, 40, 50], dtype=torch.int32, device="cuda"))
    assert torch.equal(got.logprob, want.logprob) and torch.equal(got.grad, want.grad)
    got = learner.preference_loss(c.logits, c.d_moves, torch.tensor([40, 45, 20], dtype=torch.int32, device="cuda"))
    assert got.logprob.tolist() == [0, 0] and (got.grad == 0).all()


def test_many_pairs_and_long_lines(learner):
    c = Case(3, 6000, 65, "f32", 0.5)
    preference_case(learner, c, (2900, 3100), beta=0.01)
    preference_case(learner, c, (3,) * 2000)


def test_gradients_against_differences(learner):
    """Both losses' gradients by central differences of the losses themselves, in 32 bits: steps of 2^-6 leave an error
    of the order of a thousandth (the third derivative's term, h^2 / 6) and the loss's own rounding over the step."""
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(12, 19, generator=gen).cuda()
    moves = torch.randint(0, 19, (12,), generator=gen, dtype=torch.int32).cuda()
    lp = learner.logprobs(x, moves).logprob
    old, ref = lp + 0.05 * torch.randn(12, generator=gen).cuda(), lp + 0.3 * torch.randn(12, generator=gen).cuda()
    adv = torch.randn(12, generator=gen).cuda()
    begin = torch.tensor([0, 4, 6, 6, 12], dtype=torch.int32, device="cuda")
    # clipped nowhere: a difference across a border is no derivative
    policy = lambda y, grad=False: learner.policy_loss(y, moves, old, adv, ref_logprob=ref, clip_low=0.9, clip_high=3.0,  # noqa: E731
                                                       kl_weight=0.3, scale=1.0, grad=grad)
    lines = lambda y, grad=False: learner.preference_loss(y, moves, begin, beta=0.5, label_smoothing=0.2, scale=1.0, grad=grad)  # noqa: E731
    h = 2.0 ** -6
    for loss in (policy, lines):
        g = loss(x, True).grad
        for r, j in [(0, int(moves[0])), (0, 3), (5, int(moves[5])), (7, 11), (11, 18), (6, 0)]:
            up, down = x.clone(), x.clone()
            up[r, j] += h
            down[r, j] -= h
            difference = (loss(up).loss.double() - loss(down).loss.double()) / (2 * h)
            allowed = h * h * 4 + 4 * 2.0 ** -24 * abs(float(loss(x).loss)) / h
            assert abs(float(difference - g[r, j])) <= allowed


def test_nothing_to_do(learner):
    x = torch.empty(0, 225, device="cuda")
    none = torch.empty(0, device="cuda")
    moves = torch.empty(0, dtype=torch.int32, device="cuda")
    assert learner.priors(x).shape == (0, 225)
    assert learner.logprobs(x, moves, entropy=True).entropy.shape == (0,)
    got = learner.policy_loss(x, moves, none, none)
    assert float(got.loss) == 0 and got.grad.shape == (0, 225)
    begin = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = learner.preference_loss(x, moves, begin)
    assert float(got.loss) == 0 and got.margin.shape == (0,)
    # pairs of empty lines: nothing is preferred, log 2 each
    got = learner.preference_loss(x, moves, torch.zeros(5, dtype=torch.int32, device="cuda"))
    assert abs(float(got.loss) - math.log(2)) <= 4 * O.U and got.margin.tolist() == [0, 0]


def test_the_same_every_time(learner):
    for rows, actions in ((3000, 225), (50, 50000), (2, 300000)):
        c = Case(4, rows, actions, "bf16", 0.5)
        old, adv, ref, weight = (torch.from_numpy(np.nan_to_num(a)).cuda() for a in columns(c))
        first = learner.policy_loss(c.logits, c.d_moves, old, adv, ref, weight, c.legal, kl_weight=0.1)
        begin = torch.tensor([0, rows // 3, rows], dtype=torch.int32, device="cuda")
        lines = learner.preference_loss(c.logits, c.d_moves, begin, legal=c.legal)
        for _ in range(3):
            again = learner.policy_loss(c.logits, c.d_moves, old, adv, ref, weight, c.legal, kl_weight=0.1)
            assert all(torch.equal(a, b) for a, b in zip(first, again))
            again = learner.preference_loss(c.logits, c.d_moves, begin, legal=c.legal)
            assert all(torch.equal(a, b) for a, b in zip(lines, again))


def test_rows_far_apart(learner):
    """Elements beyond 2^31 of a matrix."""
    stride = (1 << 31) + 11
    flat = torch.empty(2 * stride, dtype=torch.bfloat16, device="cuda")
    c = Case(6, 2, 1000, "bf16", 0.5)
    far = flat.as_strided((2, 1000), (stride, 1))
    far.copy_(c.logits)
    c.logits = far
    policy_case(learner, c, grad=far)


@pytest.mark.parametrize("rows,actions", [((1 << 21) * 16 + 5, 3), ((1 << 21) + 3, 4100)])
def test_more_rows_than_a_launch_takes(learner, rows, actions):
    """What the first and the last rows come to where a launch's blocks do not reach the end, by the same rows alone."""
    gen = torch.Generator("cuda").manual_seed(1)
    x = torch.empty(rows, actions, dtype=torch.float16, device="cuda")
    for at in range(0, rows, 1 << 19):
        x[at:at + (1 << 19)].normal_(0, 2, generator=gen)
    moves = torch.randint(0, actions, (rows,), device="cuda", generator=gen, dtype=torch.int32)
    adv = torch.randn(rows, device="cuda", generator=gen)
    ends = [slice(0, 64), slice(rows - 64, rows)]
    few = torch.cat([x[e] for e in ends]).clone()
    fewer = torch.cat([moves[e] for e in ends])
    lp = learner.logprobs(x, moves, entropy=True)
    alone = learner.logprobs(few, fewer, entropy=True)
    # (a row alone is summed in another order: two roundings of a sum whose terms are as many as the actions)
    for a, b in zip(lp, alone):
        assert (torch.cat([a[e] for e in ends]) - b).abs().max() <= (actions / 64 + 64) * O.U * 4
    begin = torch.tensor([0, rows // 2, rows], dtype=torch.int32, device="cuda")
    lines = learner.preference_loss(x, moves, begin, beta=1e-9, grad=False)
    sums = torch.stack([lp.logprob[:rows // 2].double().sum(), lp.logprob[rows // 2:].double().sum()])
    assert ((lines.logprob.double() - sums).abs() <= sums.abs() * 4 * O.U).all()
    got = learner.policy_loss(x, moves, lp.logprob, adv, scale=1.0, grad=x)  # in place: the last use of these logits
    assert (got.logprob - lp.logprob).abs().max() <= (actions / 64 + 64) * O.U * 4
    want = learner.policy_loss(few, fewer, torch.cat([lp.logprob[e] for e in ends]), torch.cat([adv[e] for e in ends]), scale=1.0)
    # nearly the same numbers, each rounded to 11 bits: a step of these apart at most
    assert ((torch.cat([x[e] for e in ends]).double() - want.grad.double()).abs() <=
            2.0 ** -24 + want.grad.double().abs() * (2.0 ** -10 + 2.0 ** -18)).all()
    # the ratios are 1 within the log-probabilities' rounding, so the loss is minus the advantages' sum
    assert abs(float(got.loss) + float(adv.double().sum())) <= float(adv.double().abs().sum()) * ((actions / 64 + 64) * O.U * 4 + 2.0 ** -22)


def test_graphs_and_streams(learner):
    """Calls captured into two graphs, replayed in turn and side by side, with eager work between; calls on a stream of
    their own."""
    c = [Case(20 + k, 300, 362, "bf16", 0.5) for k in range(2)]
    cols = [[torch.from_numpy(np.nan_to_num(a)).cuda() for a in columns(x)] for x in c]
    begin = torch.tensor([0, 100, 180, 240, 300], dtype=torch.int32, device="cuda")

    def work(k):
        old, adv, ref, weight = cols[k]
        x = c[k]
        return (learner.policy_loss(x.logits, x.d_moves, old, adv, ref, weight, x.legal, kl_weight=0.1),
                learner.preference_loss(x.logits, x.d_moves, begin, legal=x.legal),
                learner.logprobs(x.logits, x.d_moves, x.legal, entropy=True), (learner.priors(x.logits, x.legal),))

    side = [torch.cuda.Stream() for _ in range(2)]
    graphs, outs = [], []
    for k in range(2):
        side[k].wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side[k]):
            work(k)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side[k]):
            outs.append(work(k))
        graphs.append(g)

    def same(a, b):
        return all(torch.equal(x, y) for p, q in zip(a, b) for x, y in zip(p, q))

    for turn in range(4):
        for k in range(2):
            c[k].logits.add_(torch.randn(c[k].logits.shape, device="cuda").to(torch.bfloat16).nan_to_num() * 0.5)
        torch.cuda.synchronize()
        for k in range(2):
            with torch.cuda.stream(side[k]):
                graphs[k].replay()
        eager = [work(k) for k in range(2)]
        torch.cuda.synchronize()
        for k in range(2):
            assert same(outs[k], eager[k]), (turn, k)
    with torch.cuda.stream(side[0]):
        own = work(0)
    side[0].synchronize()
    assert same(own, work(0))


def test_python_refuses(learner):
    import omoknuni_small_amd as omk
    x = torch.randn(4, 225, device="cuda")
    moves = torch.zeros(4, dtype=torch.int32, device="cuda")
    f = torch.zeros(4, device="cuda")
    for bad in (x.double(), x.int()):
        with pytest.raises(TypeError):
            learner.priors(bad)
    for bad in (x[0], x.t(), x[:, ::2], x.cpu(), x[:, :0]):
        with pytest.raises(ValueError):
            learner.priors(bad)
    with pytest.raises(TypeError):
        learner.logprobs(x, moves.long())
    for bad in (moves[:3], moves.cpu(), moves[None]):
        with pytest.raises(ValueError):
            learner.logprobs(x, bad)
    for bad in (torch.zeros(4, 7, dtype=torch.int32, device="cuda"), torch.zeros(3, 8, dtype=torch.int32, device="cuda")):
        with pytest.raises(ValueError):
            learner.priors(x, legal=bad)
    with pytest.raises(TypeError):
        learner.priors(x, legal=torch.ones(4, 225, dtype=torch.bool, device="cuda"))
    with pytest.raises(TypeError):
        learner.policy_loss(x, moves, f.double(), f)
    with pytest.raises(omk.OmkError, match="reference"):
        learner.policy_loss(x, moves, f, f, kl_weight=0.1)
    with pytest.raises(omk.OmkError, match="clipped"):
        learner.policy_loss(x, moves, f, f, clip_low=-0.1)
    with pytest.raises(TypeError):
        learner.policy_loss(x, moves, f, f, grad=torch.empty(4, 225, dtype=torch.float16, device="cuda"))
    with pytest.raises(omk.OmkError, match="across"):
        wide = torch.zeros(5, 225, device="cuda")
        learner.policy_loss(wide[:4], moves, f, f, grad=wide[1:])
    with pytest.raises(ValueError):
        learner.preference_loss(x, moves, torch.zeros(4, dtype=torch.int32, device="cuda"))
    with pytest.raises(omk.OmkError, match="label_smoothing"):
        learner.preference_loss(x, moves, torch.zeros(3, dtype=torch.int32, device="cuda"), label_smoothing=0.7)
