"""Host-side mirror of the C ABI in include/omk_learn.h: what lies between a search and the network that it asks.

From the network's logits to the priors of an expansion (Learner.priors, Batch.expand_logits), and from the moves that a
search played to the gradient by the logits (Learner.policy_loss, Learner.preference_loss) and the step of the weights
(AdamW).  All of it works on torch tensors that are on the learner's device, on the stream that is torch's current one
there when a call is made, and waits for nothing.  Every call goes through libomk_forest.so; there is no host fallback.
Import torch before anything here or in forest.py loads that library: the two then share one HIP runtime (a torch that brings its
own and comes second finds no GPU; Learner says so).

A gradient by the logits is handed on to the network that made them: `logits.backward(got.grad)`.  That is the only way back:
results carry no history of their own (neither requires_grad nor forward-mode tangents), whatever the logits carry.
"""
import array
import collections
import ctypes as C
import operator

import numpy as np

from .forest import _check, load_library

EXPORTS = [
    "omk_learner_create", "omk_learner_destroy", "omk_learner_set_stream", "omk_learner_get_stream", "omk_learner_sync",
    "omk_policy_work", "omk_policy_priors", "omk_policy_logprobs", "omk_policy_loss_work", "omk_policy_loss",
    "omk_preference_loss_work", "omk_preference_loss",
    "omk_adamw_create", "omk_adamw_destroy", "omk_adamw_step", "omk_adamw_set_steps", "omk_adamw_get_steps",
]

_VP, _I32, _I64, _F64 = C.c_void_p, C.c_int32, C.c_int64, C.c_double


class _Rows(C.Structure):
    _fields_ = [("d_logits", _VP), ("row_stride", _I64), ("rows", _I64), ("actions", _I32), ("type", _I32),
                ("d_legal", _VP), ("legal_stride", _I64)]


class _Samples(C.Structure):
    _fields_ = [("d_moves", _VP), ("d_old_logprob", _VP), ("d_advantage", _VP), ("d_ref_logprob", _VP),
                ("d_weight", _VP)]


class _PolicyParams(C.Structure):
    _fields_ = [("clip_low", _F64), ("clip_high", _F64), ("kl_weight", _F64), ("scale", _F64)]


class _PolicyOut(C.Structure):
    _fields_ = [("d_loss", _VP), ("d_grad", _VP), ("grad_stride", _I64), ("d_logprob", _VP), ("d_kl", _VP)]


class _PreferenceParams(C.Structure):
    _fields_ = [("beta", _F64), ("label_smoothing", _F64), ("scale", _F64)]


class _PreferenceOut(C.Structure):
    _fields_ = [("d_loss", _VP), ("d_grad", _VP), ("grad_stride", _I64), ("d_margin", _VP), ("d_line_logprob", _VP),
                ("zero_rest", _I32)]


class _AdamTensor(C.Structure):
    _fields_ = [("n", _I64), ("d_param", _VP), ("d_copy", _VP), ("d_m", _VP), ("d_v", _VP), ("d_m_scale", _VP),
                ("d_v_scale", _VP), ("lr_scale", _F64), ("weight_decay", _F64)]


class _AdamDesc(C.Structure):
    _fields_ = [("n_tensors", _I32), ("h_tensors", C.POINTER(_AdamTensor)), ("param_type", _I32), ("grad_type", _I32),
                ("copy_type", _I32), ("state_type", _I32), ("beta1", _F64), ("beta2", _F64), ("eps", _F64),
                ("seed", C.c_uint32)]


_ARGTYPES = {
    "omk_learner_create": (_I32, _VP), "omk_learner_destroy": (_VP,), "omk_learner_set_stream": (_VP, _VP),
    "omk_learner_get_stream": (_VP, _VP), "omk_learner_sync": (_VP,),
    "omk_policy_work": (_I64, _I32), "omk_policy_priors": (_VP, _VP, _VP, _I64, _VP, _I64),
    "omk_policy_logprobs": (_VP, _VP, _VP, _VP, _VP, _VP, _I64),
    "omk_policy_loss_work": (_I64, _I32), "omk_policy_loss": (_VP, _VP, _VP, _VP, _VP, _VP, _I64),
    "omk_preference_loss_work": (_I64, _I32, _I64),
    "omk_preference_loss": (_VP, _VP, _VP, _VP, _I64, _VP, _VP, _VP, _VP, _I64),
    "omk_adamw_create": (_VP, _VP, _VP), "omk_adamw_destroy": (_VP,), "omk_adamw_step": (_VP, _VP, _F64, _VP, _VP),
    "omk_adamw_set_steps": (_VP, _I64), "omk_adamw_get_steps": (_VP, _VP),
}
_ready = None
_DTYPE = operator.attrgetter("dtype")
_F32, _BF16, _F16, _F8, _NONE = 0, 1, 2, 3, -1
_SMALL = 32768  # 128 KB.  (An allocation for the loss alone takes 1.6 us of a call of 17, until the kernels take longer than the call.)


def _library():
    global _ready
    lib = load_library()
    if lib is not _ready:
        for name in EXPORTS:
            fn = getattr(lib, name)
            fn.restype = _I64 if name.endswith("_work") else C.c_int
            fn.argtypes = _ARGTYPES[name]
        _ready = lib
    return lib


def _torch():
    import torch
    return torch


def _types():
    torch = _torch()
    return {torch.float32: _F32, torch.bfloat16: _BF16, torch.float16: _F16}


Logprobs = collections.namedtuple("Logprobs", "logprob entropy")
PolicyLoss = collections.namedtuple("PolicyLoss", "loss grad logprob kl")
PreferenceLoss = collections.namedtuple("PreferenceLoss", "loss grad margin logprob")


def pack_legal(mask):
    """A [.., actions] tensor of truth values (or numbers, 0 where an action is not legal) as [.., words] int32 masks: bit i of
    word i // 32."""
    torch = _torch()
    actions = mask.shape[-1]
    words = (actions + 31) // 32
    bits = torch.zeros(mask.shape[:-1] + (words * 32,), dtype=torch.int64, device=mask.device)
    bits[..., :actions] = mask != 0
    packed = (bits.unflatten(-1, (words, 32)) << torch.arange(32, device=mask.device)).sum(-1)
    return torch.where(packed >= 1 << 31, packed - (1 << 32), packed).to(torch.int32)


def legal_of_moves(move_begin, moves, actions):
    """The masks [n, words] uint32 (numpy) of n lists of moves, moves[move_begin[t]:move_begin[t + 1]]; moves outside the
    action space have no bit."""
    move_begin, moves = np.asarray(move_begin, np.int64), np.asarray(moves, np.int64)
    n, words = len(move_begin) - 1, (int(actions) + 31) // 32
    row = np.repeat(np.arange(n), np.diff(move_begin))
    move = moves[move_begin[0]:move_begin[-1]]
    inside = (move >= 0) & (move < actions)
    bits = np.zeros((n, words * 32), np.uint8)
    bits[row[inside], move[inside]] = 1
    return np.packbits(bits, axis=1, bitorder="little").view("<u4")


class Learner:
    """A device, and the operators on rows of logits there (omk_learner).

    Rows are positions (or tokens) and columns actions: logits [rows, actions] in float32, bfloat16 or float16 with any
    stride between rows.  `legal`: int32 masks [rows, words], or [words] for all rows alike, as pack_legal makes them (None:
    all actions are legal).  `moves`: int32 [rows], -1 where a row is padding.  See include/omk_learn.h for rows without
    a legal action and for infinite logits.
    """

    def __init__(self, device=None):
        self._h = C.c_void_p()
        import torch
        self._lib = _library()
        self._torch = torch
        if not torch.cuda.is_available():
            raise OSError("torch finds no GPU: if there is one, import torch before the first Forest or Learner is made "
                          "(a torch that brings a HIP runtime of its own has to be loaded first)")
        if device is None:
            device = torch.cuda.current_device()
        elif not isinstance(device, int):
            device = torch.device(device)
            device = torch.cuda.current_device() if device.index is None else device.index
        self.device = int(device)
        _check(self._lib.omk_learner_create(self.device, C.byref(self._h)))
        self._stream = 0
        self._types = _types()
        self._empty, self._f32, self._i32 = torch.empty, torch.float32, torch.int32
        self._place = torch.device("cuda", self.device)
        self._written = torch.autograd.graph.increment_version  # told of tensors that are written in place
        # (the address alone: the stream object of torch.cuda.current_stream costs a microsecond)
        self._raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
            lambda index: torch.cuda.current_stream(index).cuda_stream)

    def close(self):
        if self._h:
            self._lib.omk_learner_destroy(self._h)
            self._h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def sync(self):
        self._on_stream()
        _check(self._lib.omk_learner_sync(self._h))

    # ---- arguments ----

    def _on_stream(self):
        stream = self._raw_stream(self.device)
        if stream != self._stream:
            _check(self._lib.omk_learner_set_stream(self._h, stream))
            self._stream = stream

    def _rows(self, logits, legal):
        kind = self._types.get(logits.dtype)
        if kind is None:
            raise TypeError("logits of %s: float32, bfloat16 or float16 are taken" % logits.dtype)
        if logits.dim() != 2 or logits.shape[1] < 1:
            raise ValueError("logits of shape %s: [rows, actions] is wanted" % (tuple(logits.shape),))
        if logits.get_device() != self.device:
            raise ValueError("logits on %s: the learner's device is %d" % (logits.device, self.device))
        rows, actions = logits.shape
        stride, step = logits.stride()
        if step != 1 and actions > 1:
            raise ValueError("logits whose actions are %d elements apart" % step)
        if legal is None:
            return _Rows(logits.data_ptr(), stride, rows, actions, kind, None, 0), rows, actions
        words = (actions + 31) // 32
        self._same_place("legal", legal, self._i32)
        if tuple(legal.shape) not in ((rows, words), (words,)):
            raise ValueError("legal of shape %s: [%d, %d] or [%d] is wanted" % (tuple(legal.shape), rows, words, words))
        if words > 1 and legal.stride(-1) != 1:
            raise ValueError("legal whose words are %d apart" % legal.stride(-1))
        return _Rows(logits.data_ptr(), stride, rows, actions, kind, legal.data_ptr(),
                     0 if legal.dim() == 1 else legal.stride(0)), rows, actions

    def _same_place(self, name, x, dtype):
        if x.dtype != dtype:
            raise TypeError("%s of %s: %s is wanted" % (name, x.dtype, dtype))
        if x.get_device() != self.device:
            raise ValueError("%s on %s: the learner's device is %d" % (name, x.device, self.device))

    def _vector(self, name, x, n, dtype):
        if x is None:
            return None
        if x.dtype is dtype and x.get_device() == self.device and x.dim() == 1 and x.numel() == n and x.is_contiguous():
            return x.data_ptr()
        self._same_place(name, x, dtype)
        raise ValueError("%s of shape %s: %d values in a row are wanted" % (name, tuple(x.shape), n))

    def _gradient(self, grad, logits):
        if grad is True:
            return logits.new_empty(logits.shape)
        if grad is None or grad is False:
            return None
        self._same_place("grad", grad, logits.dtype)
        if grad.shape != logits.shape or (grad.shape[1] > 1 and grad.stride(1) != 1):
            raise ValueError("grad of shape %s, logits of %s" % (tuple(grad.shape), tuple(logits.shape)))
        return grad

    def _loss(self, small, at):
        """Where a loss is written: at `at` of the memory of a call's other small results, or where that is large in memory of
        its own, so that a program that keeps its losses keeps little else with them."""
        return small.as_strided((), (), at) if small.numel() <= _SMALL else self._empty((), dtype=self._f32, device=self._place)

    def _work(self, rows, actions):
        """Work space of the calls that need some for wide rows only."""
        need = self._lib.omk_policy_work(rows, actions)
        return (self._empty(need, dtype=self._torch.uint8, device=self._place), need) if need else (None, 0)

    def upload_legal(self, mask):
        """Masks of uint32 words in host memory (legal_of_moves) as `legal` takes them."""
        return self._torch.from_numpy(np.ascontiguousarray(mask).view(np.int32)).to(self._place)

    # ---- operators ----

    def priors(self, logits, legal=None, out=None):
        """Probabilities of the actions, float32 [rows, actions]: 0 where an action is not legal, and in a row that has
        no legal action."""
        r, rows, actions = self._rows(logits, legal)
        given = out is not None
        if not given:
            out, stride = self._empty((rows, actions), dtype=self._f32, device=self._place), actions
        else:
            self._same_place("out", out, self._f32)
            if tuple(out.shape) != (rows, actions) or (actions > 1 and out.stride(1) != 1):
                raise ValueError("out of shape %s: [%d, %d] is wanted" % (tuple(out.shape), rows, actions))
            stride = out.stride(0)
        work, need = self._work(rows, actions)
        self._on_stream()
        _check(self._lib.omk_policy_priors(self._h, C.byref(r), out.data_ptr(), stride,
                                           None if work is None else work.data_ptr(), need))
        if given:
            self._written(out)
        return out

    def logprobs(self, logits, moves=None, legal=None, entropy=False):
        """Logprobs(logprob, entropy), float32 [rows] each: the log-probability of the moves (None without moves; 0 for
        a move outside the action space, -inf for one that is not legal) and, if wanted, the entropy of the rows."""
        r, rows, actions = self._rows(logits, legal)
        d_moves = self._vector("moves", moves, rows, self._i32)
        lp = None if moves is None else self._empty(rows, dtype=self._f32, device=self._place)
        ent = self._empty(rows, dtype=self._f32, device=self._place) if entropy else None
        work, need = self._work(rows, actions)
        self._on_stream()
        _check(self._lib.omk_policy_logprobs(self._h, C.byref(r), d_moves, None if lp is None else lp.data_ptr(),
                                             None if ent is None else ent.data_ptr(),
                                             None if work is None else work.data_ptr(), need))
        return Logprobs(lp, ent)

    def policy_loss(self, logits, moves, old_logprob, advantage, ref_logprob=None, weight=None, legal=None, clip_low=0.2,
                    clip_high=0.2, kl_weight=0.0, scale=None, grad=True):
        """Clipped policy loss with a KL term towards a reference policy, and its gradient by the logits.

        old_logprob, advantage, ref_logprob, weight: float32 [rows].  scale None: 1 / rows.  grad: True for a new tensor,
        False for none, or the tensor to write (the logits themselves are allowed).  Returns PolicyLoss(loss (one
        value), grad, logprob [rows], kl [rows])."""
        r, rows, actions = self._rows(logits, legal)
        f32 = self._f32
        samples = _Samples(self._vector("moves", moves, rows, self._i32), self._vector("old_logprob", old_logprob, rows, f32),
                           self._vector("advantage", advantage, rows, f32),
                           self._vector("ref_logprob", ref_logprob, rows, f32), self._vector("weight", weight, rows, f32))
        params = _PolicyParams(clip_low, clip_high, kl_weight, 1.0 / max(rows, 1) if scale is None else scale)
        g = self._gradient(grad, logits)
        need = self._lib.omk_policy_loss_work(rows, actions)
        # one allocation for what is small: log-probabilities, kl, the loss, and the work space behind them
        behind = (2 * rows + 4) // 4 * 4
        small = old_logprob.new_empty(behind + (need + 3) // 4)
        at = small.data_ptr()
        loss = self._loss(small, 2 * rows)
        out = _PolicyOut(loss.data_ptr(), None if g is None else g.data_ptr(), 0 if g is None else g.stride(0), at,
                         at + 4 * rows)
        self._on_stream()
        _check(self._lib.omk_policy_loss(self._h, C.byref(r), C.byref(samples), C.byref(params), C.byref(out),
                                         at + 4 * behind, need))
        if g is grad and g is not None:
            self._written(g)
        view = small.as_strided
        return PolicyLoss(loss, g, view((rows,), (1,), 0), view((rows,), (1,), rows))

    def preference_loss(self, logits, moves, line_begin, ref_logprob=None, legal=None, beta=0.1, label_smoothing=0.0,
                        scale=None, grad=True):
        """Loss of pairs of lines of play, the first of a pair preferred to the second, and its gradient by the logits.

        Line s is rows line_begin[s] .. line_begin[s + 1] - 1 (int32 [2 * pairs + 1]; lines 2k and 2k + 1 are a pair);
        ref_logprob: float32 [2 * pairs], the lines' log-probabilities under the reference policy (grad=False on its
        logits gives them).  scale None: 1 / pairs.  grad: as in policy_loss; rows of no line are left as they are (a
        new tensor has zeros there).  Returns PreferenceLoss(loss, grad, margin [pairs], logprob [2 * pairs])."""
        r, rows, actions = self._rows(logits, legal)
        f32 = self._f32
        if line_begin.dim() != 1 or line_begin.shape[0] % 2 != 1:
            raise ValueError("line_begin of shape %s: two lines a pair and the end" % (tuple(line_begin.shape),))
        lines = line_begin.shape[0] - 1
        pairs = lines // 2
        d_begin = self._vector("line_begin", line_begin, lines + 1, self._i32)
        d_moves = self._vector("moves", moves, rows, self._i32)
        d_ref = self._vector("ref_logprob", ref_logprob, lines, f32)
        params = _PreferenceParams(beta, label_smoothing, 1.0 / max(pairs, 1) if scale is None else scale)
        g = self._gradient(grad, logits)
        need = self._lib.omk_preference_loss_work(rows, actions, pairs)
        behind = (3 * pairs + 4) // 4 * 4
        small = self._empty(behind + (need + 3) // 4, dtype=f32, device=self._place)
        at = small.data_ptr()
        loss = self._loss(small, 3 * pairs)
        out = _PreferenceOut(loss.data_ptr(), None if g is None else g.data_ptr(), 0 if g is None else g.stride(0), at,
                             at + 4 * pairs, grad is True)
        self._on_stream()
        _check(self._lib.omk_preference_loss(self._h, C.byref(r), d_moves, d_begin, pairs, d_ref, C.byref(params),
                                             C.byref(out), at + 4 * behind, need))
        if g is grad and g is not None:
            self._written(g)
        view = small.as_strided
        return PreferenceLoss(loss, g, view((pairs,), (1,), 0), view((lines,), (1,), pairs))


class AdamW:
    """AdamW over many tensors at once (omk_adamw), stepped in place by one launch for every 256 of them.

    params: contiguous tensors of one type on the learner's device; they stay where they are while the optimizer lives.  (Also of
    four dimensions: weights and gradients in a channels-last layout are refused.)
    copies: 16-bit tensors that take the rounded parameters with every step (32-bit parameters only).  grad_type: the
    gradients' type (None: the parameters').  states: "f32", or "f8" for moments in 8 bits with a scale for every 256
    elements.  weight_decay, lr_scale: one value, or one for every tensor.

    The moments of all tensors lie in one buffer each, every tensor's at a multiple of 256 elements (self.starts).
    """

    def __init__(self, learner, params, copies=None, grad_type=None, states="f32", betas=(0.9, 0.999), eps=1e-8,
                 weight_decay=0.01, lr_scale=1.0, seed=0):
        torch = _torch()
        self._lib, self.learner, self._h = _library(), learner, C.c_void_p()
        self.params = list(params)
        self.copies = None if copies is None else list(copies)
        n = len(self.params)
        if n == 0:
            raise ValueError("no parameters")
        if states not in ("f32", "f8"):
            raise ValueError("states %r: 'f32' or 'f8'" % (states,))
        if self.copies is not None and len(self.copies) != n:
            raise ValueError("%d copies of %d parameters" % (len(self.copies), n))
        kinds = learner._types
        self.param_type = self.params[0].dtype
        self.grad_type = grad_type or self.param_type
        copy_type = None if self.copies is None else self.copies[0].dtype
        for t in (self.param_type, self.grad_type) + (() if copy_type is None else (copy_type,)):
            if t not in kinds:
                raise TypeError("tensors of %s: float32, bfloat16 or float16 are taken" % t)
        for name, tensors, dtype in (("params", self.params, self.param_type), ("copies", self.copies or [], copy_type)):
            for x, p in zip(tensors, self.params):
                learner._same_place(name, x, dtype)
                if not x.is_contiguous() or x.numel() != p.numel():
                    raise ValueError("%s of shape %s: contiguous tensors are wanted, copies as large as theirs" %
                                     (name, tuple(x.shape)))
        decay = [weight_decay] * n if np.isscalar(weight_decay) else list(weight_decay)
        lr_scale = [lr_scale] * n if np.isscalar(lr_scale) else list(lr_scale)
        if len(decay) != n or len(lr_scale) != n:
            raise ValueError("%d values of weight_decay and %d of lr_scale for %d tensors" % (len(decay), len(lr_scale), n))
        self.starts, at = [], 0
        for p in self.params:
            self.starts.append(at)
            at += (p.numel() + 255) // 256 * 256
        device = self.params[0].device
        self.states = states
        kind = torch.float32 if states == "f32" else torch.float8_e4m3fn
        self.m, self.v = (torch.zeros(at, dtype=torch.float32, device=device).to(kind) for _ in range(2))
        self.m_scale = self.v_scale = None
        if states == "f8":
            self.m_scale, self.v_scale = (torch.zeros(at // 256, dtype=torch.float32, device=device) for _ in range(2))
        tensors = (_AdamTensor * n)()
        for i, p in enumerate(self.params):
            t, start = tensors[i], self.starts[i]
            t.n, t.d_param = p.numel(), p.data_ptr()
            t.d_copy = None if self.copies is None else self.copies[i].data_ptr()
            t.d_m, t.d_v = (x.data_ptr() + start * x.element_size() for x in (self.m, self.v))
            if states == "f8":
                t.d_m_scale, t.d_v_scale = (x.data_ptr() + start // 256 * 4 for x in (self.m_scale, self.v_scale))
            t.lr_scale, t.weight_decay = float(lr_scale[i]), float(decay[i])
        desc = _AdamDesc(n, tensors, kinds[self.param_type], kinds[self.grad_type],
                         _NONE if copy_type is None else kinds[copy_type], _F32 if states == "f32" else _F8,
                         float(betas[0]), float(betas[1]), float(eps), int(seed) & 0xFFFFFFFF)
        self._sizes = [p.numel() for p in self.params]
        # what holds the version counters of all that a step writes: views share their base's
        written = [x if x._base is None else x._base for x in self.params + (self.copies or [])]
        self._written = list({id(x): x for x in written}.values())
        learner._on_stream()
        _check(self._lib.omk_adamw_create(learner._h, C.byref(desc), C.byref(self._h)))

    def close(self):
        if self._h:
            self._lib.omk_adamw_destroy(self._h)
            self._h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def step(self, grads, lr, grad_scale=None):
        """One step.  An infinite or NaN gradient stays in the moments (with 8-bit ones in its block of 256): nothing is skipped.
        grads: a contiguous tensor of grad_type for every parameter, or None where one has none (it is left
        as it is).  lr: a number, or a float32 tensor of one value on the device.  grad_scale: a float32 tensor of one
        value that gradients are multiplied by (a clipping factor, one over a loss scale)."""
        if len(grads) != len(self.params):
            raise ValueError("%d gradients of %d parameters" % (len(grads), len(self.params)))
        learner, dtype, device = self.learner, self.grad_type, self.learner.device
        T = learner._torch.Tensor
        at = None
        if not any(g is None for g in grads):
            # (a look at all tensors' sizes, then at all their devices, .. takes half of what a look at tensor after tensor does)
            if (list(map(T.numel, grads)) == self._sizes and set(map(T.get_device, grads)) == {device} and
                    all(map(T.is_contiguous, grads)) and set(map(_DTYPE, grads)) == {dtype}):
                at = list(map(T.data_ptr, grads))
        if at is None:
            at = []
            for g, n in zip(grads, self._sizes):
                if g is None:
                    at.append(0)
                elif g.dtype is dtype and g.numel() == n and g.get_device() == device and g.is_contiguous():
                    at.append(g.data_ptr())
                else:
                    raise ValueError("gradient %d: %s %s on %s: %d contiguous values of %s on device %d are wanted" %
                                     (len(at), g.dtype, tuple(g.shape), g.device, n, dtype, device))
        d_lr, number = None, 0.0
        if isinstance(lr, (int, float)):
            number = lr
        else:
            d_lr = learner._vector("lr", lr.reshape(-1), 1, learner._f32)
        d_scale = None if grad_scale is None else learner._vector("grad_scale", grad_scale.reshape(-1), 1, learner._f32)
        learner._on_stream()
        addresses = array.array("Q", at)
        _check(self._lib.omk_adamw_step(self._h, addresses.buffer_info()[0], number, d_lr, d_scale))
        # a backward pass that has saved a weight from before this step is refused by torch, as after its own optimizers' steps
        if 0 not in at:
            learner._written(self._written)
        else:
            learner._written([x for x, g in zip(self.params, at) if g])
            if self.copies:
                learner._written([x for x, g in zip(self.copies, at) if g])

    def state(self):
        """The moments, as they are held: dict(m, v) and with 8-bit states (float8_e4m3fn, v's square root) m_scale and
        v_scale, one for every 256 elements."""
        out = dict(m=self.m, v=self.v)
        if self.states == "f8":
            out.update(m_scale=self.m_scale, v_scale=self.v_scale)
        return out

    def steps(self):
        """Steps done; waits for the stream."""
        self.learner._on_stream()
        n = C.c_int64()
        _check(self._lib.omk_adamw_get_steps(self._h, C.byref(n)))
        return n.value

    def load_state(self, steps, m, v, m_scale=None, v_scale=None):
        """Takes over moments laid out as state() gives them, and the count of the steps that made them; all of it, or where
        something is refused nothing."""
        given = dict(m=m, v=v)
        if self.states == "f8":
            given.update(m_scale=m_scale, v_scale=v_scale)
        for name, mine in self.state().items():
            x = given[name]
            if x is None or x.dtype != mine.dtype or x.shape != mine.shape:
                raise ValueError("%s: %s %s is wanted" % (name, mine.dtype, tuple(mine.shape)))
        self.learner._on_stream()
        # (held to what 64 bits pass on: ctypes would cut a larger number)
        _check(self._lib.omk_adamw_set_steps(self._h, max(-1, min(int(steps), 1 << 31))))
        for name, mine in self.state().items():
            mine.copy_(given[name])
