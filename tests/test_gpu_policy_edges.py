"""Calls on rows of logits that the tables of the other tests leave out: single rows of every width, rows of which a part holds
the type's lowest value, references far from the policy, and what lies at the ends of their ranges.  Against 64 bits, with
tolerances that count what is rounded."""
import math

import numpy as np
import pytest

from tests import learn_oracle as O

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U = 2.0 ** -24  # half a step of a 32-bit float


@pytest.fixture(scope="module")
def learner():
    import omoknuni_small_amd as omk
    return omk.Learner()


def poison(learner, elements):
    """Memory of the sizes that the next calls ask for holds what is no result."""
    held = [torch.full((n,), 12345.0, device="cuda") for n in (elements, 4096, 64, 16) for _ in range(4)]
    torch.cuda.synchronize()
    del held


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("actions", [1, 2, 225, 1500, 5000, 40000, 65528, 65529, 65537, 70001, 300000])
@pytest.mark.parametrize("rows", [1, 2])
def test_a_single_row_of_any_width(learner, kind, actions, rows):
    """A row's loss is its share: -ratio * advantage where nothing is clipped.  (One row's share is the whole loss in every kernel;
    two rows' are added up by another.)"""
    gen = torch.Generator().manual_seed(actions)
    x = torch.randn(rows, actions, generator=gen).to(TYPES[kind])
    moves = torch.randint(0, actions, (rows,), generator=gen, dtype=torch.int32)
    lp = torch.log_softmax(x.double(), 1).gather(1, moves[:, None].long())[:, 0]
    old = (lp + 0.05).float()
    advantage = torch.tensor([1.5, 0.25][:rows])
    want = -(torch.exp(lp - old.double()) * advantage.double()).sum() * 0.5
    poison(learner, rows * actions)
    got = learner.policy_loss(x.cuda(), moves.cuda(), old.cuda(), advantage.cuda(), scale=0.5)
    # the loss is rounded once; a log-probability is off by what the terms of its sum are: a few roundings each
    assert abs(float(got.loss) - float(want)) <= 8 * U * abs(float(want)) + U * abs(float(want))
    p = torch.softmax(x.double(), 1)
    slope = -(torch.exp(lp - old.double()) * advantage.double()) * 0.5
    one = torch.zeros_like(p).scatter_(1, moves[:, None].long(), 1.0)
    half = {"f32": U, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}[kind]
    g = slope[:, None] * (one - p)
    # 16 roundings of a probability or of the 1 beside it, and the result's own
    off = slope.abs()[:, None] * (p + one) * 16 * U + g.abs() * half + (2.0 ** -25 if kind == "f16" else 2.0 ** -126)
    assert ((got.grad.double().cpu() - g).abs() <= off).all()


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("actions", [225, 1500, 3000, 20011, 50000, 150000])
@pytest.mark.parametrize("where", ["first half", "last half", "all but one", "all but the last", "every other thousand"])
def test_columns_of_the_lowest_value(learner, kind, actions, where):
    """Actions masked by the type's lowest finite value, as they are where no bit masks are used: probability 0, and nothing
    to the entropy."""
    rng = np.random.default_rng(actions)
    dtype = TYPES[kind]
    x = torch.from_numpy(rng.normal(0, 2, (5, actions))).to(dtype)
    j = torch.arange(actions)
    masked = {"first half": j < actions // 2, "last half": j >= actions // 2, "all but one": j != actions // 3,
              "all but the last": j < actions - 1, "every other thousand": j // 1000 % 2 == 0}[where]
    if masked.all():
        masked[7] = False
    x[1:4, masked] = torch.finfo(dtype).min
    x[3, :] = torch.finfo(dtype).min
    o = O.Rows(x.double().numpy())
    moves = torch.from_numpy(o.p.argmax(1).astype(np.int32))
    got = learner.logprobs(x.cuda(), moves.cuda(), entropy=True)
    entropy = got.entropy.double().cpu().numpy()
    assert (np.abs(entropy - o.entropy) <= o.entropy_off()).all()
    lp, _, off = o.taken(moves.numpy())
    assert (np.abs(got.logprob.double().cpu().numpy() - lp) <= off + np.abs(lp) * U).all()
    p = learner.priors(x.cuda()).double().cpu().numpy()
    assert (np.abs(p - o.p) <= o.priors_off()).all()


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,actions", [(1, 1), (37, 225), (70, 362), (9, 5000), (3, 70001)])
def test_rows_without_a_pair(learner, kind, rows, actions):
    """No line of play: the loss is 0, a new gradient is 0 everywhere, and a given one is left as it is."""
    x = torch.randn(rows, actions, device="cuda").to(TYPES[kind])
    moves = torch.zeros(rows, dtype=torch.int32, device="cuda")
    begin = torch.full((1,), 7, dtype=torch.int32, device="cuda")
    poison(learner, rows * actions)
    poison(learner, (rows * actions + 1) // 2)
    got = learner.preference_loss(x, moves, begin)
    assert float(got.loss) == 0 and got.grad.shape == x.shape and (got.grad == 0).all()
    assert got.margin.shape == (0,) and got.logprob.shape == (0,)
    assert float(learner.preference_loss(x, moves, begin, grad=False).loss) == 0
    given = torch.full_like(x, 7.0)
    assert float(learner.preference_loss(x, moves, begin, grad=given).loss) == 0 and (given == 7).all()
    # rows with gaps, through the C ABI: what lies between two rows stays
    from omoknuni_small_amd import learn
    import ctypes as C
    wide = torch.full((rows, actions + 3), 7.0, dtype=TYPES[kind], device="cuda")
    loss = torch.full((), 7.0, device="cuda")
    r = learn._Rows(x.data_ptr(), actions, rows, actions, learner._types[x.dtype], None, 0)
    out = learn._PreferenceOut(loss.data_ptr(), wide.data_ptr(), actions + 3, None, None, 1)
    learner._on_stream()
    rc = learn._library().omk_preference_loss(learner._h, C.byref(r), None, None, 0, None, C.byref(learn._PreferenceParams(0.1, 0.0, 1.0)),
                                              C.byref(out), None, 0)
    assert rc == 0 and float(loss) == 0 and (wide[:, :actions] == 0).all() and (wide[:, actions:] == 7).all()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("actions", [2, 225, 3000, 40000, 70001])
def test_references_near_and_far(learner, kind, actions):
    """The KL term alone (no advantage): kl = exp(d) - d - 1 and the slope exp(d) - 1 for references from where the policy is to
    ones that never play the move, and ones that nearly always do."""
    ds = np.array([0, 1e-4, -1e-4, 1e-3, -1e-3, 0.01, -0.01, 0.015, 0.017, -0.24, 0.24, -0.26, 0.26, 1, -1, -3, -10, -1e3, -1e5, -1e9, -3e38, -np.inf, 5, 20])
    rng = np.random.default_rng(actions)
    x = torch.from_numpy(rng.normal(0, 1, (len(ds), actions))).to(TYPES[kind])
    o = O.Rows(x.double().numpy())
    moves = rng.integers(0, actions, len(ds)).astype(np.int32)
    lp, _, off = o.taken(moves)
    ref = (lp + ds).astype(np.float32)
    d = ref.astype(np.float64) - lp
    zero = torch.zeros(len(ds), device="cuda")
    got = learner.policy_loss(x.cuda(), torch.from_numpy(moves).cuda(), torch.from_numpy(lp.astype(np.float32)).cuda(), zero,
                              ref_logprob=torch.from_numpy(ref).cuda(), kl_weight=0.5, scale=2.0)
    slope, kl = -np.expm1(d), np.expm1(d) - d
    kl[np.abs(d) < 1e-5] = (d * d / 2)[np.abs(d) < 1e-5]
    # both are worked out in 64 bits from a log-probability that is `off` off, and rounded once (the slope, a probability and their
    # product: three times)
    kl_off = np.abs(slope) * off + np.exp(d) * off ** 2 + kl * U * 1.01
    mine = got.kl.double().cpu().numpy()
    with np.errstate(invalid="ignore"):
        assert ((np.abs(mine - kl) <= kl_off) | (mine == kl)).all()
    assert np.isinf(mine[21]) and float(got.loss) == np.inf
    g, g_off = o.gradient(moves, slope, np.exp(d) * off + np.abs(slope) * 4 * U, kind)
    mine = got.grad.double().cpu().numpy()
    assert (np.abs(mine - g) <= g_off).all()
    # without the infinite one the loss is the divergences' sum
    keep = [i for i in range(len(ds)) if i != 21]
    put = lambda a: torch.from_numpy(a[keep]).cuda()  # noqa: E731
    got = learner.policy_loss(x[keep].cuda(), put(moves), put(lp.astype(np.float32)), zero[:len(keep)], ref_logprob=put(ref), kl_weight=1e-30,
                              scale=2.0)
    want = 2e-30 * kl[keep].sum()
    assert abs(float(got.loss) - want) <= 2 * U * want


WIDTHS = [2, 31, 225, 362, 1500, 5000, 20011, 40000, 70001]  # of every kernel that holds, streams or cuts rows


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("actions", WIDTHS)
def test_log_probabilities_are_as_exact_as_their_terms(learner, kind, actions):
    """How far log-probabilities are off before they are rounded, seen through the divergence from a reference close by:
    kl(d + t) = kl(d) + (exp(d) - 1) t + ..

    Logits are multiples of 1/16, so that differences are exact.  A term exp(x - m) is then off by 4e-8 (rms) and 5e-9 on the mean (two
    roundings of the instruction and of the correction); sums are exact beside that.  So t has a mean of 5e-9 and a spread of
    4e-8 sqrt(sum p^2); six of these are allowed, and the divergence's own rounding, U d/2."""
    rng = np.random.default_rng(actions)
    rows = max(8, min(400, 2000000 // actions))
    x = np.round(rng.normal(0, 2, (rows, actions)).clip(-7, 7) * 16) / 16
    if actions > 1000:
        x[0] = -3.0
        x[0, actions // 2:] = 2.5  # the largest logits all in one half: the other's sums are relative to another maximum
    o = O.Rows(x)
    moves = rng.integers(0, actions, rows).astype(np.int32)
    lp, _, _ = o.taken(moves)
    ref = (lp + 0.01).astype(np.float32)
    d = ref.astype(np.float64) - lp
    zero = torch.zeros(rows, device="cuda")
    got = learner.policy_loss(torch.from_numpy(x).to(TYPES[kind]).cuda(), torch.from_numpy(moves).cuda(), zero, zero,
                              ref_logprob=torch.from_numpy(ref).cuda())
    kl = np.expm1(d) - d
    off = 5e-9 + 6 * 4e-8 * np.sqrt((o.p ** 2).sum(1)) * (o.p.max(1) < 1)
    t = (got.kl.double().cpu().numpy() - kl) / np.expm1(d)
    assert (np.abs(t) <= off + U * np.abs(d)).all(), np.abs(t / off).max()


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("actions", WIDTHS)
def test_rows_that_are_all_but_decided(learner, kind, actions):
    """One action far above the others: log-probability -log(1 + (n - 1) exp(-gap)) and entropy keep their digits beside the 1.

    Every other term is off by a step of the exponential (2 U) and the correction's rounding (U), the sum of them by nothing, and
    the result is rounded (U)."""
    gaps = np.array([3.0, 8.0, 11.0, 13.0, 15.0, 17.0])
    x = np.zeros((len(gaps), actions))
    at = np.arange(len(gaps)) * (actions - 1) // (len(gaps) - 1)
    x[np.arange(len(gaps)), at] = gaps
    rest = (actions - 1) * np.exp(-gaps)
    got = learner.logprobs(torch.from_numpy(x).to(TYPES[kind]).cuda(), torch.from_numpy(at.astype(np.int32)).cuda(), entropy=True)
    lp = -np.log1p(rest)
    assert (np.abs(got.logprob.double().cpu().numpy() - lp) <= 4.1 * U * np.abs(lp)).all()
    entropy = np.log1p(rest) + rest * gaps / (1 + rest)
    # the second part adds terms of one size up in 32 bits: n/64 of them one after another at most, then lanes and wavefronts
    off = 4.1 * U * np.log1p(rest) + (actions / 64 + 24) * U * rest * gaps / (1 + rest) + 2 * U * entropy
    assert (np.abs(got.entropy.double().cpu().numpy() - entropy) <= off).all()
    lines = learner.preference_loss(torch.from_numpy(x).to(TYPES[kind]).cuda(), torch.from_numpy(at.astype(np.int32)).cuda(),
                                    torch.tensor([0, 1, 6], dtype=torch.int32, device="cuda"), grad=False).logprob.double().cpu().numpy()
    want = np.array([lp[0], lp[1:].sum()])
    assert (np.abs(lines - want) <= 4.1 * U * np.abs(want)).all()


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("actions", WIDTHS)
@pytest.mark.parametrize("which", ["policy", "lines"])
def test_gradients_of_rows_that_are_all_but_decided(learner, kind, actions, which):
    """The gradient at a move that is nearly certain is slope * (1 - p): as exact as the others, to which it adds up to 0.

    1 - p is good to two steps of the exponential and a rounding (3 U) and the product is rounded, the slope before it; the other
    actions' probabilities are off by 3 U, the sum's rounding, a reciprocal to a step (2 U) and three products."""
    gaps = np.array([3.0, 8.0, 11.0, 13.0, 15.0, 17.0])
    x = np.zeros((len(gaps), actions))
    at = np.arange(len(gaps)) * (actions - 1) // (len(gaps) - 1)
    x[np.arange(len(gaps)), at] = gaps
    e = np.exp(-gaps)
    rest = (actions - 1) * e
    dx, moves = torch.from_numpy(x).to(TYPES[kind]).cuda(), torch.from_numpy(at.astype(np.int32)).cuda()
    scale = 4096.0  # (in 16 bits with a narrow range these would be next to its end)
    lp = -np.log1p(rest)
    if which == "policy":
        got = learner.policy_loss(dx, moves, torch.from_numpy(lp.astype(np.float32)).cuda(), torch.ones(len(gaps), device="cuda"), scale=scale)
        slope = -scale * np.exp(lp - lp.astype(np.float32))
    else:
        got = learner.preference_loss(dx, moves, torch.tensor([0, 2, 6], dtype=torch.int32, device="cuda"), beta=0.5, scale=scale)
        u = 0.5 * (lp[:2].sum() - lp[2:].sum())
        slope = -0.5 * scale / (1 + np.exp(u)) * np.where(np.arange(6) < 2, 1, -1)
    grad = got.grad.double().cpu().numpy()
    half, tiny = {"f32": (U, 2.0 ** -126), "bf16": (2.0 ** -8, 2.0 ** -126), "f16": (2.0 ** -11, 2.0 ** -25)}[kind]
    # (the pairs' slope is worked out in 32 bits: expf, a sum, a quotient, two products)
    slope_rel = U if which == "policy" else 16 * U
    want = slope * rest / (1 + rest)
    assert (np.abs(grad[np.arange(6), at] - want) <= np.abs(want) * (4.1 * U + slope_rel + half) + tiny).all()
    grad[np.arange(6), at] = np.nan
    want = np.where(np.isnan(grad), np.nan, (-slope * e / (1 + rest))[:, None])
    # (by the form without the correction where terms are computed again: x U and 2.2e-8 x more)
    off = np.abs(want) * (10 * U + 2 * gaps[:, None] * U + slope_rel + half) + tiny
    assert ((np.abs(grad - want) <= off) | np.isnan(want)).all()


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("actions", [225, 3000, 40000, 70001])
def test_ratios_beyond_the_range(learner, kind, actions):
    """A ratio that no 32-bit number holds: illegal actions' gradients are 0 all the same, and nothing is NaN."""
    import omoknuni_small_amd as omk
    gen = torch.Generator().manual_seed(actions)
    mask = torch.rand(4, actions, generator=gen) < 0.5
    mask[:, 3] = True
    x = torch.randn(4, actions, generator=gen).to(TYPES[kind]).masked_fill(~mask, float("nan")).cuda()
    moves = torch.full((4,), 3, dtype=torch.int32, device="cuda")
    old = torch.tensor([-300.0, -math.inf, -3.0, -300.0], device="cuda")
    adv = torch.tensor([-1.0, -1.0, -1.0, 1.0], device="cuda")  # (the last is clipped)
    got = learner.policy_loss(x, moves, old, adv, legal=omk.pack_legal(mask).cuda(), scale=1.0)
    assert float(got.loss) == math.inf
    assert not got.grad.isnan().any() and (got.grad[~mask.cuda()] == 0).all() and (got.grad[3] == 0).all()
    assert (got.grad[:2, 3].float() >= (60000 if kind == "f16" else 1e38)).all()


@pytest.mark.parametrize("beta,smoothing", [(0.5, 0.1), (0.3, 0.25), (0.1, 0.0), (0.7, 0.5)])
def test_slopes_of_pairs_next_to_their_least_loss(learner, beta, smoothing):
    """Two actions alike, so that log-probabilities are -log 2 exactly (to 2^-53): the margin is what the references make it, and
    the gradient slope / 2.  Each result is rounded to 32 bits once; the gradient's slope and its product with 1/2 too."""
    best = math.log((1 - smoothing) / smoothing) if smoothing else 5.0
    deltas = np.concatenate([best + np.array([1e-2, 1e-4, -1e-5, 1e-6, -3e-7, 0.1]), np.array([0.0, 1.0, -2.0, 30.0, -30.0, 300.0, -300.0])])
    pairs = len(deltas)
    ref = np.zeros((pairs, 2), np.float32)
    ref[:, 0] = -math.log(2.0) - deltas / beta
    u = beta * ((-3 * math.log(2.0) - ref[:, 0].astype(np.float64)) + 2 * math.log(2.0))
    begin = torch.cat([torch.tensor([5 * k, 5 * k + 3], dtype=torch.int32) for k in range(pairs)] + [torch.tensor([5 * pairs], dtype=torch.int32)])
    x = torch.zeros(5 * pairs, 2, device="cuda")
    moves = torch.zeros(5 * pairs, dtype=torch.int32, device="cuda")
    got = learner.preference_loss(x, moves, begin.cuda(), ref_logprob=torch.from_numpy(ref.reshape(-1)).cuda(), beta=beta,
                                  label_smoothing=smoothing, scale=1.0)
    margin = got.margin.double().cpu().numpy()
    assert (np.abs(margin - u) <= U * np.abs(u) + 1e-15).all()
    with np.errstate(over="ignore"):
        slope = -beta * ((1 - smoothing) / (1 + np.exp(u)) - smoothing / (1 + np.exp(-u)))
        loss = ((1 - smoothing) * np.logaddexp(0, -u) + smoothing * np.logaddexp(0, u)).sum()
    grad = got.grad.double().cpu().numpy().reshape(pairs, 5, 2)
    sign = np.array([1, 1, 1, -1, -1])[None, :, None] * np.array([0.5, -0.5])[None, None]
    want = slope[:, None, None] * sign
    assert (np.abs(grad - want) <= 2.1 * U * np.abs(want) + 2.0 ** -126 + 1e-15).all()
    assert abs(float(got.loss) - loss) <= 2.1 * U * loss


@pytest.mark.parametrize("rows,actions", [(3, 7), (4096, 7), (10000, 7), (100000, 7), (2000, 70001)])
def test_a_kept_loss_keeps_little(learner, rows, actions):
    """The memory that a loss holds on to, once all else of its call is gone."""
    x = torch.zeros(rows, actions, device="cuda", dtype=torch.bfloat16)
    moves, f = torch.zeros(rows, dtype=torch.int32, device="cuda"), torch.zeros(rows, device="cuda")
    got = learner.policy_loss(x, moves, f - math.log(actions), f + 1, grad=False)
    assert got.loss.untyped_storage().nbytes() <= 131072 and abs(float(got.loss) + 1) < 1e-5
    got = learner.preference_loss(x, moves, torch.tensor([0, rows // 2, rows], dtype=torch.int32, device="cuda"), scale=0.0, grad=False)
    assert got.loss.untyped_storage().nbytes() <= 131072 and float(got.loss) == 0
