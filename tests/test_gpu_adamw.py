"""AdamW over many tensors at once against the formula in 64 bits, and its 8-bit states against the same arithmetic made
step by step in numpy."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HALF_STEP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
TINY = {"f32": 2.0 ** -149, "bf16": 2.0 ** -133, "f16": 2.0 ** -25}
B1, B2, EPS, LR = 0.9, 0.999, 1e-8, 1e-2


@pytest.fixture(scope="module")
def learner():
    import omoknuni_small_amd as omk
    return omk.Learner()


def mix(h):
    h = np.asarray(h, np.uint64) & 0xFFFFFFFF
    h ^= h >> 16
    h = h * 0x7FEB352D & 0xFFFFFFFF
    h ^= h >> 15
    h = h * 0x846CA68B & 0xFFFFFFFF
    return h ^ (h >> 16)


E4M3 = np.array([(c & 7) / 8 * 2.0 ** -6 if c < 8 else (1 + (c & 7) / 8) * 2.0 ** ((c >> 3) - 7) for c in range(127)])


def to_8_bits(x, random16):
    """Codes (from their definition: the neighbours in the list of all codes) and the scale of one block of float32."""
    f = np.float32
    top = np.abs(x).max()
    if not top > 2.0 ** -100:
        return np.zeros(len(x), np.int64), f(0)
    y = np.minimum(np.abs(x) * (f(1) / top * f(448)), f(448))
    shifted = np.where(y < f(2.0 ** -6), y + f(2.0 ** -6), y).astype(np.float64) - np.where(y < f(2.0 ** -6), 2.0 ** -6, 0)
    below = np.searchsorted(E4M3, shifted, side="right") - 1
    step = np.append(np.diff(E4M3), 32.0)[below]
    # 2^-16 of a step is what the random number counts in; the place between the codes is kept to 2^-20
    place = np.floor((shifted - E4M3[below]) / step * 2 ** 20)
    return below + (place + random16 * 16 >= 2 ** 20), top * f(1.0 / 448.0)


def random_of(seed, t, unit, n):
    key = mix(mix(seed ^ (t * 0x9E3779B1 & 0xFFFFFFFF)) ^ np.uint64(unit))
    return mix((key + np.arange(n, dtype=np.uint64) * np.uint64(0x9E3779B1)) & np.uint64(0xFFFFFFFF))


class Plain:
    """The optimizer in numpy: moments in 32 bits or coded, the parameter's step in 64 bits beside how far the GPU's
    may be from it."""

    def __init__(self, sizes, states, seed, decay, lr_scale):
        self.sizes, self.states, self.seed, self.decay, self.lr_scale, self.t = sizes, states, seed, decay, lr_scale, 0
        self.m = [np.zeros(n, np.float32) for n in sizes]
        self.r = [np.zeros(n, np.float32) for n in sizes]  # sqrt(v), as it is held with 8 bits
        self.v = [np.zeros(n, np.float32) for n in sizes]
        self.codes = {}

    def step(self, p, grads, lr, grad_scale=np.float32(1)):
        """p: float64 of what the parameters held.  Returns (new parameters in 64 bits, off) per tensor."""
        f = np.float32
        self.t += 1
        out, unit = [], 0
        for i, n in enumerate(self.sizes):
            units = (n + 255) // 256
            if grads[i] is None:
                out.append((p[i], np.zeros(n)))
                unit += units
                continue
            g = grads[i].astype(f) * grad_scale
            v_old = self.r[i] * self.r[i] if self.states == "f8" else self.v[i]
            m = self.m[i] * f(B1) + g * f(1 - B1)
            v = v_old * f(B2) + (g * g) * f(1 - B2)
            root = np.sqrt(v)
            rate = lr * self.lr_scale[i] / (1 - B1 ** self.t)
            down = np.sqrt(v.astype(np.float64)) / math.sqrt(1 - B2 ** self.t) + EPS
            with np.errstate(invalid="ignore", divide="ignore"):
                update = rate * m.astype(np.float64) / down
            shrink = lr * self.lr_scale[i] * self.decay[i]
            new = p[i] * (1 - shrink) - update
            # a rounded rate and its product (2 U), the root's half step, a rounded factor and its product (3 U), a sum (U),
            # a reciprocal that is good to a step (2 U) and its product (U): 9 U of the update; the decay's product and
            # both differences: 2 U of what they give
            off = np.abs(update) * 9 * U + np.abs(p[i] * shrink) * 3 * U + (np.abs(p[i]) + np.abs(new)) * 2 * U
            out.append((new, off))
            self.m[i], self.v[i] = m, v
            if self.states == "f8":
                self.m[i], self.r[i] = m.copy(), root.copy()
                for b in range(units):
                    at = slice(256 * b, min(n, 256 * b + 256))
                    random = random_of(self.seed, self.t, unit + b, at.stop - at.start)
                    for name, x, bits in (("m", m[at], random & 0xFFFF), ("v", root[at], random >> 16)):
                        code, scale = to_8_bits(x, bits.astype(np.float64))
                        if name == "v":
                            y = np.minimum(np.abs(x) * (f(1) / x.max() * f(448)), f(448)) if scale else np.zeros_like(x)
                            code = np.maximum(code, y > 0)
                        value = E4M3[code].astype(f) * scale
                        if name == "m":
                            self.m[i][at] = np.where(x < 0, -value, value)
                        else:
                            self.r[i][at] = value
                        self.codes[i, b, name] = (code, scale)
            unit += units
        return out


def setup(learner, sizes, param="f32", grad="f32", copy=None, states="f32", seed=77, shift=0):
    import omoknuni_small_amd as omk
    rng = np.random.default_rng(len(sizes) * 31 + sum(sizes))
    params = []
    for n in sizes:  # `shift`: addresses with the alignment of the type only
        flat = torch.zeros(n + shift, dtype=TYPES[param], device="cuda")
        flat[shift:] = torch.from_numpy(rng.normal(0, 0.1, n)).to(TYPES[param])
        params.append(flat[shift:])
    copies = None if copy is None else [torch.zeros(n + shift, dtype=TYPES[copy], device="cuda")[shift:] for n in sizes]
    decay = [0.05 if i % 2 else 0.0 for i in range(len(sizes))]
    lr_scale = [1.0 if i % 3 else 0.5 for i in range(len(sizes))]
    opt = omk.AdamW(learner, params, copies=copies, grad_type=TYPES[grad], states=states, betas=(B1, B2), eps=EPS,
                    weight_decay=decay, lr_scale=lr_scale, seed=seed)
    return opt, Plain(sizes, states, seed, decay, lr_scale), rng


def gradients(rng, sizes, grad, shift=0):
    out = []
    for i, n in enumerate(sizes):
        flat = torch.zeros(n + shift, dtype=TYPES[grad])
        flat[shift:] = torch.from_numpy(rng.normal(0, 10.0 ** (i % 5 - 3), n) * (rng.random(n) < 0.9)).to(TYPES[grad])
        out.append(flat.cuda()[shift:])
    return out


def check(opt, plain, sizes, before, grads, param, lr=LR, scale=np.float32(1)):
    want = plain.step(before, [None if g is None else g.float().cpu().numpy() for g in grads], lr, scale)
    for i, n in enumerate(sizes):
        got, (new, off) = opt.params[i].double().cpu().numpy(), want[i]
        assert (np.abs(got - new) <= off + np.abs(new) * HALF_STEP[param] + TINY[param]).all(), i
        if opt.copies is not None and grads[i] is not None:
            assert torch.equal(opt.copies[i], opt.params[i].to(opt.copies[i].dtype)), i
        start = opt.starts[i]
        state = {k: v.cpu() for k, v in opt.state().items()}
        if opt.states == "f32":
            assert (state["m"][start:start + n].numpy() == plain.m[i]).all(), i
            assert (state["v"][start:start + n].numpy() == plain.v[i]).all(), i
            continue
        for name, held in (("m", plain.m[i]), ("v", plain.r[i])):
            scales = np.repeat(state[name + "_scale"].numpy()[start // 256:start // 256 + (n + 255) // 256], 256)[:n]
            assert (state[name][start:start + n].float().numpy() * scales == held).all(), (i, name)


SIZES = [(1,), (255, 256, 257), (3, 2048, 1, 2049, 700, 5000), (70000, 5)]


@pytest.mark.parametrize("states", ["f32", "f8"])
@pytest.mark.parametrize("sizes", SIZES, ids=str)
@pytest.mark.parametrize("param,grad,copy", [("f32", "f32", None), ("f32", "bf16", "bf16"), ("f32", "f16", "f16"),
                                             ("f32", "f32", "bf16"), ("bf16", "bf16", None), ("f16", "f16", None),
                                             ("bf16", "f32", None), ("f16", "f32", None)])
def test_steps(learner, states, sizes, param, grad, copy):
    for shift in (0, 1):
        opt, plain, rng = setup(learner, sizes, param, grad, copy, states, shift=shift)
        for _ in range(3):
            before = [p.double().cpu().numpy() for p in opt.params]
            g = gradients(rng, sizes, grad, shift)
            opt.step(g, lr=LR)
            check(opt, plain, sizes, before, g, param)
        assert opt.steps() == 3


@pytest.mark.parametrize("states", ["f32", "f8"])
def test_tensors_without_gradients_and_many_of_them(learner, states):
    """More tensors than travel with one launch, some without a gradient, some empty; a scale and a rate from the device."""
    sizes = [(7 * i) % 600 for i in range(600)]
    opt, plain, rng = setup(learner, sizes, states=states)
    scale, lr = torch.tensor([0.25], device="cuda"), torch.tensor(0.02, device="cuda")
    for turn in range(2):
        before = [p.double().cpu().numpy() for p in opt.params]
        g = gradients(rng, sizes, "f32")
        g = [None if (i + turn) % 7 == 0 else x for i, x in enumerate(g)]
        opt.step(g, lr=lr, grad_scale=scale)
        check(opt, plain, sizes, before, g, "f32", lr=float(np.float32(0.02)), scale=np.float32(0.25))
    assert opt.steps() == 2


def test_extreme_gradients_in_8_bits(learner):
    """Blocks of nothing, of one value, of values too small to keep, of a range that codes cannot span, and of no numbers:
    the last stays in its block."""
    sizes = (256 * 6,)
    opt, plain, rng = setup(learner, sizes, states="f8")
    g = np.zeros(sizes[0], np.float32)
    g[256] = 3.0
    g[512:768] = 1e-36
    g[768:1024] = (10.0 ** rng.uniform(-12, 3, 256)).astype(np.float32)
    g[1024:1280] = rng.normal(0, 1, 256)
    for _ in range(3):
        before = [p.double().cpu().numpy() for p in opt.params]
        x = torch.from_numpy(g).cuda()
        opt.step([x], lr=LR)
        check(opt, plain, sizes, before, [x], "f32")
    # every second moment that is not 0 is held as more than 0, so that no step divides by eps alone
    held = opt.state()["v"].float()
    assert (held[768:1024] > 0).all() and (held[:256] == 0).all()
    good = opt.state()["m"].float().clone()
    x[1300] = math.nan
    x[1030] = math.inf
    opt.step([x], lr=LR)
    bad = [b for b in range(6) if opt.params[0][256 * b:256 * b + 256].isnan().any()]
    assert bad == [4, 5]
    scales = opt.state()["m_scale"]
    assert scales[:4].isfinite().all() and not scales[4:].isfinite().any()
    assert good.isfinite().all()


def test_rounding_is_fair(learner):
    """The mean of many codes of one value is that value: 2^16 elements between two codes, an eighth of the way (their sum is binomial:
    six standard deviations)."""
    n = 1 << 16
    x = torch.full((n,), 1.0 + 1.0 / 64, device="cuda")
    x[::256] = 448.0
    import omoknuni_small_amd as omk
    p = torch.zeros(n, device="cuda")
    opt = omk.AdamW(learner, [p], states="f8", betas=(0.0, 0.0), seed=5)
    opt.step([x], lr=0.0)
    inside = torch.ones(n, dtype=torch.bool, device="cuda")
    inside[::256] = False
    for name in ("m", "v"):
        codes = opt.state()[name].float()[inside]
        up = float((codes == 1.125).float().mean())
        assert ((codes == 1.0) | (codes == 1.125)).all()
        assert abs(up - 0.125) <= 6 * math.sqrt(0.125 * 0.875 / n)


@pytest.mark.parametrize("states", ["f32", "f8"])
def test_a_captured_step_counts(learner, states):
    sizes = (300, 2500)
    opt, plain, rng = setup(learner, sizes, states=states, copy="bf16")
    g = gradients(rng, sizes, "f32")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        opt.step(g, lr=LR)
    assert opt.steps() == 0
    for turn in range(3):
        before = [p.double().cpu().numpy() for p in opt.params]
        for x, y in zip(g, gradients(rng, sizes, "f32")):
            x.copy_(y)
        graph.replay()
        check(opt, plain, sizes, before, g, "f32")
        before = [p.double().cpu().numpy() for p in opt.params]
        opt.step(g, lr=LR)
        check(opt, plain, sizes, before, g, "f32")
    assert opt.steps() == 6


@pytest.mark.parametrize("states", ["f32", "f8"])
def test_state_taken_over(learner, states):
    import omoknuni_small_amd as omk
    sizes = (1000, 70)
    opt, plain, rng = setup(learner, sizes, states=states)
    for _ in range(5):
        opt.step(gradients(rng, sizes, "f32"), lr=LR)
    other = omk.AdamW(learner, [p.clone() for p in opt.params], states=states, betas=(B1, B2), eps=EPS,
                      weight_decay=plain.decay, lr_scale=plain.lr_scale, seed=77)
    other.load_state(steps=opt.steps(), **opt.state())
    g = gradients(rng, sizes, "f32")
    opt.step(g, lr=LR)
    other.step(g, lr=LR)
    assert all(torch.equal(a, b) for a, b in zip(opt.params, other.params))
    for a, b in zip(opt.state().values(), other.state().values()):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    with pytest.raises(ValueError):
        other.load_state(steps=1, m=opt.m[:-1], v=opt.v)


def test_refusals(learner):
    import omoknuni_small_amd as omk
    p = [torch.zeros(10, device="cuda"), torch.zeros(4, 5, device="cuda")]
    for bad in (dict(states="f16"), dict(copies=[p[0].bfloat16()]), dict(weight_decay=[0.1])):
        with pytest.raises(ValueError):
            omk.AdamW(learner, p, **bad)
    with pytest.raises(TypeError):
        omk.AdamW(learner, [p[0], p[1].bfloat16()])
    with pytest.raises(TypeError):
        omk.AdamW(learner, [p[0].double()])
    with pytest.raises(ValueError):
        omk.AdamW(learner, [p[0].cpu()])
    with pytest.raises(ValueError):
        omk.AdamW(learner, [])
    with pytest.raises(ValueError):
        omk.AdamW(learner, [p[1].t()])
    with pytest.raises(omk.OmkError, match="betas"):
        omk.AdamW(learner, p, betas=(1.0, 0.9))
    with pytest.raises(omk.OmkError, match="other 16-bit"):
        omk.AdamW(learner, [p[0].bfloat16()], grad_type=torch.float16)
    opt = omk.AdamW(learner, p)
    for bad in ([p[0]], [p[0], p[0]], [p[0], p[1].t()], [p[0].cpu(), p[1]], [p[0].half(), p[1]]):
        with pytest.raises(ValueError):
            opt.step(bad, lr=0.1)
    with pytest.raises(omk.OmkError, match="lr"):
        opt.step(p, lr=math.inf)
    assert opt.steps() == 0
