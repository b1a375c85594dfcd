"""The operators between a search and the network that it asks, as cases that can be timed.

  priors      a batch of leaves is answered with logits over the action space; the search wants probabilities of the
              legal moves, in 32 bits
  logprobs    the log-probability of the move taken at every position (what a later update compares with) and the
              entropy of the policy there
  policy      one update from searched positions: clipped policy loss with a KL term towards a reference policy, and
              its gradient by the logits
  preference  pairs of lines of play, the first of each preferred to the second: the loss of their paired
              log-ratios, and its gradient by the logits
  adamw       the step of the network's weights that follows: AdamW over all its tensors, moments in 32 bits or in 8

Rows are positions (or tokens), columns actions.  Legal moves are bit masks, 32 actions a word, as a forest's `legal` is.
Boards are those of the benchmark configurations: Gomoku 15x15 with 225 actions, Go with 362, chess with at most 218;
wider rows stand for action spaces the size of a vocabulary.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CLIP_LOW, CLIP_HIGH, KL_WEIGHT = 0.2, 0.25, 0.04
PREFERENCE_BETA, SMOOTHING = 0.1, 0.05
LR, BETA1, BETA2, EPS, DECAY = 2e-4, 0.9, 0.999, 1e-8, 0.01
STEPS_DONE = 1000  # the optimizer's count before the step that is timed
SEED = 20240607  # of the 8-bit states' rounding


def _rows(name, kind, rows, actions, dtype, **options):
    c = dict(kind=kind, rows=rows, actions=actions, type=dtype, legal=0.0, weights=False, reference=True)
    c.update(options)
    return dict(c, name=name) if name else c


def _lines(name, pairs, shortest, longest, actions, dtype, **options):
    c = dict(kind="preference", pairs=pairs, shortest=shortest, longest=longest, actions=actions, type=dtype, legal=0.0)
    c.update(options)
    return dict(c, name=name) if name else c


def _adamw(name, width, blocks, states, **options):
    c = dict(kind="adamw", width=width, blocks=blocks, states=states, param="f32", grad="f32", copy="none")
    c.update(options)
    return dict(c, name=name) if name else c


def listed():
    return [
        # the leaf of a game against a person: one Go position, nothing but latency counts
        _rows("priors_go_1", "priors", 1, 362, "f32", legal=0.6),
        # the leaves of 4096 descents at once
        _rows("priors_go_4096", "priors", 4096, 362, "bf16", legal=0.6),
        # what a frozen policy gives the moves of 2049 positions over a very wide, odd action space
        _rows("logprobs_wide", "logprobs", 2049, 50001, "f16"),
        # an update on the positions of one chess game
        _rows("policy_chess_90", "policy", 90, 218, "f32", legal=0.2),
        # an update on a batch of Go positions
        _rows("policy_go_4096", "policy", 4096, 362, "bf16", legal=0.6, weights=True),
        # all positions that a generation of Gomoku games left, in one pass
        _rows("policy_gomoku_epoch", "policy", 131072, 225, "f32", legal=0.5, weights=True),
        # rows as wide as a vocabulary, where memory's rate is what counts
        _rows("policy_wide", "policy", 8192, 32768, "bf16"),
        # pairs of Gomoku lines that part after an opening, one preferred by the search
        _lines("preference_gomoku", 24, 5, 60, 225, "bf16", legal=0.5),
        # long lines over a wide action space
        _lines("preference_wide", 16, 96, 512, 32768, "bf16"),
        # the step of a small network, weights and gradients in 32 bits: many short tensors
        _adamw("adamw_small", 64, 6, "f32"),
        # the step of a large one: gradients from a bf16 backward pass, weights in 32 bits with a bf16 copy to compute with
        _adamw("adamw_large", 512, 20, "f32", grad="bf16", copy="bf16"),
        # the same with both moments in 8 bits
        _adamw("adamw_large_8bit", 512, 20, "f8", grad="bf16", copy="bf16"),
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


MOST_ELEMENTS = 8192 * 32768


def draw(rng):
    kind = rng.choice(["priors", "logprobs", "policy", "policy", "preference", "preference", "adamw", "adamw"])
    if kind == "adamw":
        blocks = rng.randint(1, 20)
        param = rng.choice(["f32", "f32", "bf16"])
        return _adamw(None, _log_uniform(rng, 16, 512), blocks, rng.choice(["f32", "f8"]), param=param,
                      grad=rng.choice(["f32", "bf16"]) if param == "f32" else "bf16",
                      copy=rng.choice(["none", "bf16"]) if param == "f32" else "none")
    board = rng.random() < 0.5
    actions = rng.choice([218, 225, 362]) if board else _log_uniform(rng, 2, 65536)
    legal = round(rng.uniform(0.1, 0.9), 2) if board or rng.random() < 0.3 else 0.0
    dtype = rng.choice(["f32", "bf16", "f16"])
    if kind == "preference":
        longest = _log_uniform(rng, 2, 512)
        pairs = max(1, min(_log_uniform(rng, 1, 256), MOST_ELEMENTS // (4 * longest * actions)))
        return _lines(None, pairs, rng.randint(1, longest), longest, actions, dtype, legal=legal)
    rows = max(1, min(_log_uniform(rng, 1, 131072), MOST_ELEMENTS // (2 * actions)))
    return _rows(None, kind, rows, actions, dtype, legal=legal, weights=rng.random() < 0.5,
                 reference=rng.random() < 0.7)


# ---- what a user's program has in hand ----

def _generator(seed):
    return torch.Generator("cuda").manual_seed(int(seed) * 7919 + 13)


def _pack(mask):
    """[rows, actions] truth values as words of 32 actions, the lowest bit the first."""
    rows, actions = mask.shape
    words = (actions + 31) // 32
    padded = torch.zeros(rows, words * 32, dtype=torch.int64, device=mask.device)
    padded[:, :actions] = mask
    packed = (padded.view(rows, words, 32) << torch.arange(32, device=mask.device)).sum(-1)
    return torch.where(packed >= 1 << 31, packed - (1 << 32), packed).to(torch.int32)


def _policy_rows(case, rows, gen, left_out):
    """Logits, legal moves, the move taken in every row (drawn from the policy; -1 where there is none) and its
    log-probability."""
    actions, dtype = case["actions"], TYPES[case["type"]]
    logits = torch.empty(rows, actions, dtype=dtype, device="cuda")
    moves = torch.empty(rows, dtype=torch.int32, device="cuda")
    logprob = torch.empty(rows, device="cuda")
    legal = None
    if case["legal"]:
        mask = torch.rand(rows, actions, device="cuda", generator=gen) < case["legal"]
        mask[torch.arange(rows, device="cuda"), torch.randint(actions, (rows,), device="cuda", generator=gen)] = True
        if left_out:  # games that are over: no move is legal
            mask[torch.rand(rows, device="cuda", generator=gen) < 0.01] = False
        legal = _pack(mask)
    piece = max(1, (1 << 26) // actions)
    for at in range(0, rows, piece):
        x = torch.randn(min(piece, rows - at), actions, device="cuda", generator=gen) * 2.0
        logits[at:at + piece] = x
        x = logits[at:at + piece].float()
        if legal is not None:
            x = x.masked_fill(~mask[at:at + piece], -math.inf)
        noise = torch.rand(x.shape, device="cuda", generator=gen).clamp_(1e-7, 1.0 - 1e-7)
        best = (x - torch.log(-torch.log(noise))).argmax(1)
        moves[at:at + piece] = best.to(torch.int32)
        logprob[at:at + piece] = x.gather(1, best[:, None])[:, 0] - torch.logsumexp(x, 1)
    none = ~torch.isfinite(logprob)
    if left_out:  # positions that were played at random or belong to padding
        none |= torch.rand(rows, device="cuda", generator=gen) < 0.03
    moves[none] = -1
    return dict(logits=logits, legal=legal, moves=moves), torch.where(none, torch.zeros_like(logprob), logprob)


def _shapes(case):
    """Elements of every tensor of a tower of residual blocks on a 19x19 board with a policy and a value head, and
    whether its weights decay."""
    w, cells, actions = case["width"], 361, 362
    sizes = [(17 * 9 * w, True), (w, False), (w, False)]
    for _ in range(2 * case["blocks"]):
        sizes += [(9 * w * w, True), (w, False), (w, False)]
    sizes += [(2 * w, True), (2, False), (2 * cells * actions, True), (actions, False)]
    sizes += [(w, True), (1, False), (cells * 256, True), (256, False), (256, True), (1, False)]
    return sizes


def _lengths(case):
    """Lengths of the lines, from the shortest to the longest."""
    last = 2 * case["pairs"] - 1
    return [case["shortest"] + (case["longest"] - case["shortest"]) * k // last for k in range(last + 1)]


def _network(case, gen):
    """Weights, gradients and moments, every tensor at a multiple of 256 elements of one buffer."""
    starts, at = [], 0
    for n, _ in _shapes(case):
        starts.append(at)
        at += (n + 255) // 256 * 256
    real = torch.zeros(at, dtype=torch.bool, device="cuda")
    decay = torch.zeros(at, device="cuda")
    size = torch.zeros(at, device="cuda")
    for (n, decays), start in zip(_shapes(case), starts):
        real[start:start + n] = True
        decay[start:start + n] = DECAY if decays else 0.0
        # gradients of a layer are as large as its size makes them
        size[start:start + n] = 1e-2 / math.sqrt(n)
    normal = lambda: torch.randn(at, device="cuda", generator=gen) * real  # noqa: E731
    s = dict(starts=starts, decay=decay, param=(normal() * 0.05).to(TYPES[case["param"]]),
             grad=(normal() * size).to(TYPES[case["grad"]]))
    if case["copy"] != "none":
        s["copy"] = s["param"].to(TYPES[case["copy"]])
    m = normal() * size * 0.3
    v = (0.2 + normal().square()) * size.square() * real
    if case["states"] == "f32":
        s.update(m=m, v=v)
    else:
        for name, x in (("m", m), ("v", v.sqrt())):
            blocks = x.view(-1, 256)
            scale = blocks.abs().amax(1) * (1.0 / 448.0)
            s[name] = (blocks / scale.clamp_min(1e-30)[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(-1)
            s[name + "_scale"] = scale
    return s


def _inputs(case, seed):
    gen = _generator(seed)
    kind = case["kind"]
    if kind == "adamw":
        return _network(case, gen)
    if kind == "preference":
        lengths = torch.tensor(_lengths(case), device="cuda")
        lengths = lengths[torch.randperm(len(lengths), device="cuda", generator=gen)]
        begin = torch.cat([lengths.new_zeros(1), lengths.cumsum(0)]).to(torch.int32)
        s, logprob = _policy_rows(case, int(begin[-1]), gen, True)
        line = torch.repeat_interleave(torch.arange(2 * case["pairs"], device="cuda"), (begin[1:] - begin[:-1]).long())
        ref = torch.zeros(2 * case["pairs"], dtype=torch.float64, device="cuda").index_add_(0, line, logprob.double())
        noise = torch.randn(2 * case["pairs"], device="cuda", generator=gen)
        s.update(begin=begin, ref=(ref + 4.0 * noise).float())
        return s
    s, logprob = _policy_rows(case, case["rows"], gen, kind == "policy")
    if kind == "policy":
        near = lambda spread: logprob + spread * torch.randn(logprob.shape, device="cuda", generator=gen)  # noqa: E731
        s["old"] = near(0.2)
        s["ref"] = near(0.5) if case["reference"] else None
        s["advantage"] = torch.randn(logprob.shape, device="cuda", generator=gen)
        s["weight"] = torch.rand(logprob.shape, device="cuda", generator=gen) + 0.5 if case["weights"] else None
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:
        import omoknuni_small_amd as omk
        s["learner"] = omk.Learner()
        if case["kind"] == "adamw":
            views = lambda x: [x[a:a + n] for a, (n, _) in zip(s["starts"], _shapes(case))]  # noqa: E731
            s["adamw"] = omk.AdamW(s["learner"], views(s["param"]),
                                   copies=views(s["copy"]) if "copy" in s else None,
                                   grad_type=TYPES[case["grad"]], states=case["states"], betas=(BETA1, BETA2), eps=EPS,
                                   weight_decay=[DECAY if decays else 0.0 for _, decays in _shapes(case)], seed=SEED)
            s["adamw"].load_state(steps=STEPS_DONE, **{k: s[k] for k in ("m", "v", "m_scale", "v_scale") if k in s})
            s["grads"] = views(s["grad"])
    elif case["kind"] == "adamw":
        s["steps"] = STEPS_DONE
    return s


# ---- the plain forms ----

def _legal_mask(s):
    x, legal = s["logits"], s["legal"]
    if legal is None:
        return None
    bits = (legal[:, :, None] >> torch.arange(32, device=x.device, dtype=torch.int32)) & 1
    return bits.flatten(1)[:, :x.shape[1]] != 0


def _softmax(s):
    """Logits in 32 bits (-inf where a move is not legal), probabilities (0 in a row that has none), the rows' largest
    logit, sum of exponentials and whether a row has a legal move; sums in 64 bits, since a loss is compared with
    borders."""
    x = s["logits"].float()
    mask = _legal_mask(s)
    if mask is not None:
        x = torch.where(mask, x, -math.inf)
    top = x.amax(1, keepdim=True)
    some = top > -math.inf
    e = torch.exp(x - torch.where(some, top, 0.0))
    total = e.sum(1, keepdim=True, dtype=torch.float64)
    return x, e / torch.where(some, total, 1.0).float(), top, total, some[:, 0]


def _taken(s, x, top, total, some):
    """Log-probability of the moves taken, in 64 bits, and the rows that count."""
    moves = s["moves"].long()
    inside = (moves >= 0) & (moves < x.shape[1])
    at = torch.where(inside, moves, 0)
    chosen = x.gather(1, at[:, None])[:, 0]
    counts = inside & some & (chosen > -math.inf)
    logp = (chosen.double() - top[:, 0].double()) - torch.log(torch.where(counts, total[:, 0], 1.0))
    return torch.where(counts, logp, 0.0), counts, at


def _gradient(s, p, at, by_logprob):
    """d loss / d logits of rows whose loss has the derivative `by_logprob` by the move's log-probability."""
    by_logprob = by_logprob.float()[:, None]
    grad = -by_logprob * p
    grad.scatter_add_(1, at[:, None], by_logprob)
    return grad.to(s["logits"].dtype)


def _priors(s):
    return _softmax(s)[1]


def _logprobs(s):
    x, p, top, total, some = _softmax(s)
    logp, counts, at = _taken(s, x, top, total, some)
    centred = torch.where(p > 0, p * (x - top), 0.0).sum(1, dtype=torch.float64)
    entropy = torch.where(some, torch.log(total[:, 0]) - centred, 0.0)
    return logp.float(), entropy.float()


def _policy(s):
    x, p, top, total, some = _softmax(s)
    logp, counts, at = _taken(s, x, top, total, some)
    advantage = s["advantage"].double()
    shift = logp - s["old"].double()
    ratio = torch.exp(shift)
    low, high = 1.0 - CLIP_LOW, 1.0 + CLIP_HIGH
    clipped = torch.where(advantage > 0, ratio > high, ratio < low)
    row = -torch.minimum(ratio * advantage, ratio.clamp(low, high) * advantage)
    by_logprob = torch.where(clipped, 0.0, -advantage * ratio)
    kl = torch.zeros_like(logp)
    if s["ref"] is not None:
        d = s["ref"].double() - logp
        kl = torch.expm1(d) - d
        row = row + KL_WEIGHT * kl
        by_logprob = by_logprob - KL_WEIGHT * torch.expm1(d)
    weight = torch.where(counts, s["weight"].double() if s["weight"] is not None else 1.0, 0.0) / len(logp)
    loss = (weight * row).sum()
    return dict(loss=loss.float(), grad=_gradient(s, p, at, weight * by_logprob), logprob=logp.float(),
                kl=torch.where(counts, kl, 0.0).float())


def _preference(s):
    x, p, top, total, some = _softmax(s)
    logp, counts, at = _taken(s, x, top, total, some)
    begin, lines = s["begin"].long(), len(s["begin"]) - 1
    line = torch.repeat_interleave(torch.arange(lines, device=x.device), begin[1:] - begin[:-1], output_size=len(logp))
    sums = torch.zeros(lines, dtype=torch.float64, device=x.device).index_add_(0, line, logp)
    gain = sums - s["ref"].double()
    margin = PREFERENCE_BETA * (gain[0::2] - gain[1::2])
    softplus = lambda t: torch.clamp(t, min=0) + torch.log1p(torch.exp(-t.abs()))  # noqa: E731
    pairs = lines // 2
    loss = ((1.0 - SMOOTHING) * softplus(-margin) + SMOOTHING * softplus(margin)).sum() / pairs
    by_first = -PREFERENCE_BETA / pairs * ((1.0 - SMOOTHING) / (1.0 + torch.exp(margin)) -
                                           SMOOTHING / (1.0 + torch.exp(-margin)))
    by_line = torch.stack([by_first, -by_first], 1).flatten()
    by_logprob = torch.where(counts, by_line[line], 0.0)
    return dict(loss=loss.float(), grad=_gradient(s, p, at, by_logprob), margin=margin.float(), logprob=sums.float())


def _mix(h):
    """Mixes the bits of 32-bit numbers, held in 64: xorshifts and products with odd constants."""
    h = h ^ (h >> 16)
    h = (h * 0x7FEB352D) & 0xFFFFFFFF
    h = h ^ (h >> 15)
    h = (h * 0x846CA68B) & 0xFFFFFFFF
    return h ^ (h >> 16)


def _to_8_bits(x, random):
    """e4m3 codes of blocks of 256 values and their scales: the block's largest magnitude becomes 448, and what lies
    between two codes goes up with the probability of its place between them.  `random`: 16 random bits a value."""
    top = x.abs().amax(1, keepdim=True)
    kept = top > 2.0 ** -100
    inverse = torch.where(kept, top, 1.0).reciprocal() * 448.0
    y = torch.where(kept, x.abs() * inverse, 0.0).clamp(max=448.0)
    small = y < 2.0 ** -6  # codes below are evenly spaced, as they are in the binade above that
    bits = torch.where(small, y + 2.0 ** -6, y).view(torch.int32)
    code = ((bits + (random << 4).to(torch.int32)) >> 20) - 960 - 8 * small.to(torch.int32)
    return code, torch.where(kept, top, 0.0)[:, 0] * (1.0 / 448.0), y


def _adamw_step(s):
    case = s["case"]
    s["steps"] += 1
    t = s["steps"]
    g = s["grad"].float()
    if case["states"] == "f32":
        m, v = s["m"], s["v"]
    else:
        m = (s["m"].float().view(-1, 256) * s["m_scale"][:, None]).view(-1)
        v = (s["v"].float().view(-1, 256) * s["v_scale"][:, None]).view(-1).square()
    m = m * BETA1 + g * (1.0 - BETA1)
    v = v * BETA2 + (g * g) * (1.0 - BETA2)
    root = v.sqrt()
    p = s["param"].float()
    p = p - p * (s["decay"] * LR)
    p = p - m * (LR / (1.0 - BETA1 ** t)) / (root * (1.0 / math.sqrt(1.0 - BETA2 ** t)) + EPS)
    s["param"].copy_(p)
    if "copy" in s:
        s["copy"].copy_(p)
    if case["states"] == "f32":
        s["m"], s["v"] = m, v
    else:
        blocks = torch.arange(len(s["m_scale"]), device=g.device)
        key = _mix(_mix(torch.tensor(SEED, device=g.device) ^ ((t * 0x9E3779B1) & 0xFFFFFFFF)) ^ blocks)
        random = _mix((key[:, None] + torch.arange(256, device=g.device) * 0x9E3779B1) & 0xFFFFFFFF)
        code, s["m_scale"], _ = _to_8_bits(m.view(-1, 256), random & 0xFFFF)
        code = code | (m.view(-1, 256) < 0).to(torch.int32) << 7
        s["m"] = code.to(torch.uint8).view(torch.float8_e4m3fn).view(-1)
        code, s["v_scale"], y = _to_8_bits(root.view(-1, 256), random >> 16)
        code = torch.maximum(code, (y > 0).to(torch.int32))  # what is not nothing is not kept as nothing
        s["v"] = code.to(torch.uint8).view(torch.float8_e4m3fn).view(-1)
    return {k: s[k] for k in ("param", "copy", "m", "v", "m_scale", "v_scale") if k in s}


# ---- the calls of a user's program ----

def _own(s):
    case, learner = s["case"], s["learner"]
    kind = case["kind"]
    if kind == "adamw":
        s["adamw"].step(s["grads"], lr=LR)
        out = {k: s[k] for k in ("param", "copy") if k in s}
        out.update(s["adamw"].state())
        return out
    if kind == "priors":
        return learner.priors(s["logits"], legal=s["legal"])
    if kind == "logprobs":
        got = learner.logprobs(s["logits"], s["moves"], legal=s["legal"], entropy=True)
        return got.logprob, got.entropy
    if kind == "policy":
        got = learner.policy_loss(s["logits"], s["moves"], s["old"], s["advantage"], ref_logprob=s["ref"],
                                  weight=s["weight"], legal=s["legal"], clip_low=CLIP_LOW, clip_high=CLIP_HIGH,
                                  kl_weight=KL_WEIGHT if s["ref"] is not None else 0.0, scale=1.0 / case["rows"])
        return dict(loss=got.loss, grad=got.grad, logprob=got.logprob, kl=got.kl)
    got = learner.preference_loss(s["logits"], s["moves"], s["begin"], ref_logprob=s["ref"], legal=s["legal"],
                                  beta=PREFERENCE_BETA, label_smoothing=SMOOTHING, scale=1.0 / case["pairs"])
    return dict(loss=got.loss, grad=got.grad, margin=got.margin, logprob=got.logprob)


def run(state):
    if own:
        return _own(state)
    plain = dict(priors=_priors, logprobs=_logprobs, policy=_policy, preference=_preference, adamw=_adamw_step)
    return plain[state["case"]["kind"]](state)


# ---- what a pass cannot do without ----

def work(case):
    kind = case["kind"]
    width = {"f32": 4, "bf16": 2, "f16": 2, "f8": 1, "none": 0}
    if kind == "adamw":
        n = sum(size for size, _ in _shapes(case))
        blocks = sum((size + 255) // 256 for size, _ in _shapes(case))
        scales = 16 * blocks if case["states"] == "f8" else 0
        return {"bytes": n * (2 * width[case["param"]] + width[case["grad"]] + width[case["copy"]] +
                              4 * width[case["states"]]) + scales, "flops": 15.0 * n}
    rows = case["rows"] if kind != "preference" else sum(_lengths(case))
    elements = rows * case["actions"]
    mask = rows * ((case["actions"] + 31) // 32) * 4 if case["legal"] else 0
    read = elements * width[case["type"]] + mask
    if kind == "priors":
        return {"bytes": read + 4 * elements, "flops": 4.0 * elements}
    if kind == "logprobs":
        return {"bytes": read + 12 * rows, "flops": 5.0 * elements}
    columns = 5 + case["reference"] + case["weights"] if kind == "policy" else 1
    return {"bytes": read + elements * width[case["type"]] + 4 * columns * rows, "flops": 6.0 * elements}


# ---- the definition, in 64 bits, row by row ----

def _exact_rows(s, at, upto):
    """Probabilities and log-probabilities of a few rows: log-softmax over the legal actions."""
    x = s["logits"][at:upto].double()
    if s["legal"] is not None:
        words = s["legal"][at:upto].long() & 0xFFFFFFFF
        j = torch.arange(x.shape[1], device=x.device)
        x[((words[:, j // 32] >> (j % 32)) & 1) == 0] = -math.inf
    return x - torch.logsumexp(x, 1, keepdim=True)  # NaN in a row without a legal action


def _exact_all(s):
    rows, actions = s["logits"].shape
    step = max(1, (1 << 25) // actions)
    for at in range(0, rows, step):
        yield at, min(rows, at + step)


def _exact_taken(s):
    rows, actions = s["logits"].shape
    taken = torch.zeros(rows, dtype=torch.float64, device="cuda")
    entropy = torch.zeros(rows, dtype=torch.float64, device="cuda")
    for at, upto in _exact_all(s):
        logp = _exact_rows(s, at, upto)
        p = logp.exp()
        entropy[at:upto] = torch.nan_to_num(-(p * logp.masked_fill(p == 0, 0.0)).sum(1), nan=0.0)
        move = s["moves"][at:upto].long()
        counted = (move >= 0) & (move < actions)
        got = logp[torch.arange(upto - at, device="cuda"), torch.where(counted, move, 0)]
        taken[at:upto] = torch.where(counted, got, math.nan)
    return taken, entropy


def _exact_gradient(s, by_logprob):
    grad = torch.zeros(s["logits"].shape, dtype=torch.float64, device="cuda")
    for at, upto in _exact_all(s):
        piece = -_exact_rows(s, at, upto).exp()
        r = torch.nonzero(s["moves"][at:upto] >= 0)[:, 0]
        piece[r, s["moves"][at:upto][r].long()] += 1.0
        c = by_logprob[at:upto, None]
        grad[at:upto] = torch.where(c == 0, torch.zeros_like(piece), piece * c)
    return grad


def exact(case, seed):
    s = _inputs(case, seed)
    kind = case["kind"]
    if kind == "priors":
        p = torch.empty(s["logits"].shape, dtype=torch.float64, device="cuda")
        for at, upto in _exact_all(s):
            p[at:upto] = torch.nan_to_num(_exact_rows(s, at, upto).exp(), nan=0.0)
        return p
    if kind == "adamw":
        t = STEPS_DONE + 1
        g, p, m, v = (s[k].double() for k in ("grad", "param", "m", "v"))
        if case["states"] == "f8":
            m = m * s["m_scale"].double().repeat_interleave(256)
            v = (v * s["v_scale"].double().repeat_interleave(256)) ** 2
        m = BETA1 * m + (1 - BETA1) * g
        v = BETA2 * v + (1 - BETA2) * g * g
        p = p * (1 - LR * s["decay"].double())
        p -= LR * (m / (1 - BETA1 ** t)) / (torch.sqrt(v / (1 - BETA2 ** t)) + EPS)
        out = dict(param=p, copy=p, m=m, v=v)
        if case["states"] == "f8":  # codes are rounded at random; their scales have a value
            out.update(m=None, v=None, m_scale=m.view(-1, 256).abs().amax(1) / 448,
                       v_scale=v.sqrt().view(-1, 256).amax(1) / 448)
        return {k: x for k, x in out.items() if k in s}
    taken, entropy = _exact_taken(s)
    if kind == "logprobs":
        return torch.nan_to_num(taken, nan=0.0), entropy
    counted = torch.isfinite(taken)
    if kind == "policy":
        weight = (s["weight"].double() if s["weight"] is not None else torch.ones_like(taken)) / case["rows"]
        a = s["advantage"].double()
        r = (taken - s["old"].double()).exp()
        bounded = r.clip(1 - CLIP_LOW, 1 + CLIP_HIGH)
        row = torch.maximum(-r * a, -bounded * a)
        slope = torch.where(-r * a >= -bounded * a, -a * r, torch.zeros_like(a))
        kl = torch.zeros_like(taken)
        if s["ref"] is not None:
            u = (s["ref"].double() - taken).exp()
            kl = u - 1 - (s["ref"].double() - taken)
            row, slope = row + KL_WEIGHT * kl, slope + KL_WEIGHT * (1 - u)
        zero = torch.zeros_like(taken)
        return dict(loss=torch.where(counted, weight * row, zero).sum(),
                    grad=_exact_gradient(s, torch.where(counted, weight * slope, zero)),
                    logprob=torch.where(counted, taken, zero), kl=torch.where(counted, kl, zero))
    ends = s["begin"].tolist()
    taken = torch.where(counted, taken, torch.zeros_like(taken))
    sums = torch.stack([taken[a:b].sum() for a, b in zip(ends, ends[1:])])
    gain = sums - s["ref"].double()
    u = PREFERENCE_BETA * (gain[0::2] - gain[1::2])
    pairs = case["pairs"]
    loss = -((1 - SMOOTHING) * torch.nn.functional.logsigmoid(u) + SMOOTHING * torch.nn.functional.logsigmoid(-u)).mean()
    slope = -PREFERENCE_BETA / pairs * ((1 - SMOOTHING) * torch.sigmoid(-u) - SMOOTHING * torch.sigmoid(u))
    by_logprob = torch.zeros_like(taken)
    for k, (a, b) in enumerate(zip(ends, ends[1:])):
        by_logprob[a:b] = slope[k // 2] * (1 if k % 2 == 0 else -1)
    by_logprob = torch.where(counted, by_logprob, torch.zeros_like(taken))
    return dict(loss=loss, grad=_exact_gradient(s, by_logprob), margin=u, logprob=sums)
