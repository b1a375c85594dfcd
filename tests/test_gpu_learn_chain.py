"""The operators between a search and its network together, as a self-play program uses them: priors from logits when
leaves are expanded, log-probabilities of the moves that the search chose, both losses' gradients through the network,
and the step of its weights, whose answers the next search takes."""
import numpy as np
import pytest

from tests import learn_oracle as O
from tests.test_gpu_policy_rows import near

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

ACTIONS, FEATURES, HIDDEN = 41, 24, 32


@pytest.fixture(scope="module")
def learner():
    import omoknuni_small_amd as omk
    return omk.Learner()


def roots_only(n):
    return dict(N=np.zeros(n, np.int32), W=np.zeros(n, np.float32), P=np.ones(n, np.float32), VL=np.zeros(n, np.int32),
                child_begin=np.zeros(n, np.int32), child_count=np.zeros(n, np.int32), action=np.full(n, -1, np.int32))


def offers(nodes, games=0):
    """The legal moves of every leaf, a function of the node; some leaves are terminal, but none of the first `games`."""
    begin, moves = [0], []
    for node in nodes:
        r = np.random.default_rng(int(node) * 7919 + 5)
        k = 0 if r.random() < 0.15 and node >= games else int(r.integers(1, ACTIONS + 1))
        moves.extend(r.choice(ACTIONS, size=k, replace=False).tolist())
        begin.append(len(moves))
    return np.array(begin, np.int32), np.array(moves, np.int32)


def features(nodes):
    return torch.from_numpy(np.stack([np.random.default_rng(int(n) + 1).normal(0, 1, FEATURES) for n in nodes])).float().cuda()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("widening", [None, (2.0, 0.5)])
def test_expansion_from_logits(learner, dtype, widening):
    """The children that expand_ex makes from the same probabilities in 64 bits, with priors as near to these as the
    operator's are; a mask with every leaf's moves, terminal leaves among them."""
    import omoknuni_small_amd as omk
    games = 40
    f = omk.Forest.from_soa(roots_only(games), capacity=40_000)
    b = omk.Batch(f, 2 * games, 16)
    b.set_roots(np.repeat(np.arange(games, dtype=np.int32), 2))
    gen = torch.Generator("cuda").manual_seed(1)
    for _ in range(3):
        b.select(omk.SelectParams())
        _, _, leaf, _ = b.read()
        before = f.download_structure()["child_count"]
        begin, moves = offers(leaf)
        logits = (torch.randn(len(leaf), ACTIONS, device="cuda", generator=gen) * 3).to(dtype)
        first = b.expand_logits(begin, moves, logits, learner, widening)
        mask = np.zeros((len(leaf), ACTIONS), bool)
        for t in range(len(leaf)):
            mask[t, moves[begin[t]:begin[t + 1]]] = True
        want = O.Rows(logits.double().cpu().numpy(), mask)
        off = want.priors_off()
        st, P = f.download_structure(), f.download()["P"]
        made = 0
        for t in range(len(leaf)):
            if first[t] < 0:
                continue
            assert before[leaf[t]] == 0 and st["child_begin"][leaf[t]] == first[t]
            kids = np.arange(first[t], first[t] + st["child_count"][leaf[t]])
            offered = moves[begin[t]:begin[t + 1]]
            assert (st["action"][kids] == offered[:len(kids)]).all() and (widening or len(kids) == len(offered))
            assert (np.abs(P[kids] - want.p[t, offered[:len(kids)]]) <= off[t, offered[:len(kids)]]).all()
            made += 1
        assert made
        b.set_values(np.linspace(-1, 1, len(leaf)).astype(np.float32))
        b.backup(3)
    with pytest.raises(ValueError):
        b.expand_logits(begin, moves, logits[:-1], learner)


class Network:
    """tanh layer and logits, in 32 bits, with a bf16 copy of the weights that the optimizer keeps."""

    def __init__(self):
        gen = torch.Generator("cuda").manual_seed(7)
        shapes = [(FEATURES, HIDDEN), (HIDDEN,), (HIDDEN, ACTIONS), (ACTIONS,)]
        self.weights = [(torch.randn(s, device="cuda", generator=gen) * 0.3).requires_grad_() for s in shapes]

    def logits(self, x):
        a, b, c, d = self.weights
        return torch.tanh(x @ a + b) @ c + d


def in_64_bits(weights, x, slope_of_logits):
    """Gradients by the weights, and sums of the magnitudes that they are sums of (what their rounding goes by)."""
    w = [p.detach().double().cpu().requires_grad_() for p in weights]
    h = torch.tanh(x.double().cpu() @ w[0] + w[1])
    (h @ w[2] + w[3]).backward(slope_of_logits)
    g, ah, ax = slope_of_logits.abs(), h.detach().abs(), x.double().cpu().abs()
    back = (g @ w[2].detach().abs().T) * (1 + ah ** 2)
    return [p.grad for p in w], [ax.T @ back, back.sum(0), ah.T @ g, g.sum(0)]


@pytest.mark.parametrize("states", ["f32", "f8"])
def test_search_learn_search(learner, states):
    import omoknuni_small_amd as omk
    games, per_game, rounds = 24, 4, 6
    net = Network()
    copies = [torch.empty(p.shape, dtype=torch.bfloat16, device="cuda") for p in net.weights]
    opt = omk.AdamW(learner, [p.detach() for p in net.weights], copies=copies, states=states, weight_decay=[0.1, 0, 0.1, 0])
    for generation in range(2):
        f = omk.Forest.from_soa(roots_only(games), capacity=60_000)
        b = omk.Batch(f, games * per_game, 24)
        b.set_roots(np.repeat(np.arange(games, dtype=np.int32), per_game))
        for _ in range(rounds):
            b.select(omk.SelectParams())
            _, _, leaf, _ = b.read()
            begin, moves = offers(leaf, games)
            with torch.no_grad():
                logits = net.logits(features(leaf))
            b.expand_logits(begin, moves, logits, learner)
            b.set_values(np.tanh(features(leaf).sum(1).cpu().numpy() / 5).astype(np.float32))
            b.backup(3)
        # the move that every game plays, what it was worth over the position, and the policy it was searched with
        N_W = f.download()
        st = f.download_structure()
        played, advantage = [], []
        for g in range(games):
            p, kids = f.action_probabilities(g, 1.0, ACTIONS)
            assert kids and abs(p.sum() - 1) < 1e-5
            move = int(p.argmax())
            child = int(st["child_begin"][g] + np.nonzero(st["action"][st["child_begin"][g]:st["child_begin"][g] + kids] == move)[0][0])
            played.append(move)
            advantage.append(-N_W["W"][child] / max(N_W["N"][child], 1) + N_W["W"][g] / max(N_W["N"][g], 1))
        begin, moves = offers(np.arange(games), games)
        from omoknuni_small_amd.learn import legal_of_moves
        masks = legal_of_moves(begin, moves, ACTIONS)
        legal = learner.upload_legal(masks)
        mask = np.unpackbits(masks.view(np.uint8), axis=1, bitorder="little")[:, :ACTIONS].astype(bool)
        x, d_moves = features(np.arange(games)), torch.tensor(played, dtype=torch.int32, device="cuda")
        adv = torch.tensor(advantage, dtype=torch.float32, device="cuda")
        with torch.no_grad():
            old = learner.logprobs(net.logits(x), d_moves, legal=legal).logprob
        assert old.isfinite().all()
        lines = torch.arange(0, games + 1, 2, dtype=torch.int32, device="cuda")  # lines of two positions
        for update in range(3):
            logits = net.logits(x)
            held = O.Rows(logits.detach().double().cpu().numpy(), mask)
            if update < 2:
                got = learner.policy_loss(logits, d_moves, old, adv, ref_logprob=old, legal=legal, kl_weight=0.1)
                want = O.policy_loss(held, np.array(played), old.double().cpu().numpy(), adv.double().cpu().numpy(),
                                     old.double().cpu().numpy(), None, 0.2, 0.2, 0.1, 1 / games)
            else:
                got = learner.preference_loss(logits, d_moves, lines, legal=legal, beta=0.5)
                want = O.preference_loss(held, np.array(played), lines.cpu().numpy(), None, 0.5, 0.0, 1 / (games // 4))
            slope, slope_off = held.gradient(np.array(played), *want["slope"], "f32")
            near(got.grad, slope, slope_off, "gradient by the logits")
            logits.backward(got.grad)
            exact, sizes = in_64_bits(net.weights, x, torch.from_numpy(slope))
            for p, g, size in zip(net.weights, exact, sizes):
                # products of three factors in 32 bits each, summed over games, actions or hidden units: as many roundings
                # as there are terms at most, and as many again for the factors' own
                allowed = 2 * (games + ACTIONS + HIDDEN + 16) * O.U * size + float(np.abs(slope_off).max()) * 50
                assert ((p.grad.double().cpu() - g).abs() <= allowed).all()
            kept = [p.detach().clone() for p in net.weights]
            opt.step([p.grad for p in net.weights], lr=3e-3)
            for p, before, copy in zip(net.weights, kept, copies):
                assert not torch.equal(p.detach(), before) and torch.equal(copy, p.detach().bfloat16())
                p.grad = None
    assert opt.steps() == 6
