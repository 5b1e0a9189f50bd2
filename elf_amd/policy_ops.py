"""The policy network's operators around its convolutions (libgoenv.so, include/goenv.h "Policy-network operators"):

* :func:`group_norm_act` -- group norm of a channels-last tensor, the residual sum and the activation of a block
* :func:`dropout`        -- dropout from a counter-based generator; the mask is never stored
* :func:`policy_logits`  -- penalties for repeated moves, biases, legal masks and a temperature on policy logits,
  as logits, log probabilities or the probabilities that ``GoEnv.sample_policy`` / ``topk_policy`` take

All of them take torch-ROCm tensors, run on torch's current stream of the tensors' device, allocate their outputs (and
nothing that outlives the call) through torch, and can be captured into a graph.  (A backward pass under capture needs leaves
no eager graph of which lives on the default stream; a call under capture with such a leaf is refused.)  What they refuse raises
:class:`elf_amd.goenv.GoEnvError`.  Gradients: once, through the backward pass of ``torch.autograd``; a tensor with a forward-mode derivative is
refused, and so is a call while torch records a trace (``torch.jit.trace``, ``make_fx``).  There is no CPU fallback.
"""
import torch
import torch.nn as nn

_native = None


def _ops():
    """The native half (csrc/policy_ops_torch.cc).  Raises if it has not been built."""
    global _native
    if _native is None:
        try:
            from . import _policy_ops
        except ImportError as e:
            raise RuntimeError("elf_amd/_policy_ops is missing: build it with `python -c 'import __graft_entry__ as g; "
                               "g.build()'`; there is no CPU fallback for the policy-network operators") from e
        _native = _policy_ops
    return _native


def group_norm_act(x, num_groups, weight=None, bias=None, eps=1e-5, act="none", slope=0.1, residual=None):
    """act(group_norm(x) * weight + bias + residual), goenv_group_norm_act.

    x: [n, c, *positions], float32, bfloat16 or float16, channels last (``memory_format=torch.channels_last``, or any
    view whose channels lie next to each other: a slice of channels, of samples).  Statistics are taken per sample
    over the positions and the c / num_groups channels of a group, in float32.  (Groups of more than some 4,000 channels
    are slow, above all their gradients.)  weight, bias: [c], float32 or x's
    type.  residual: of x's shape and type, channels last.  act: "none", "relu", "leaky_relu" (with `slope`) or
    "silu".  The result is dense and channels last, of x's type.  Gradients for x, residual, weight and bias."""
    return _ops().group_norm_act(x, num_groups, weight, bias, eps, act, slope, residual)


class GroupNormAct(nn.Module):
    """group_norm_act with a float32 weight and bias of its own; forward(x, residual=None)."""

    def __init__(self, num_groups, num_channels, eps=1e-5, act="none", slope=0.1):
        super().__init__()
        self.num_groups, self.eps, self.act, self.slope = num_groups, eps, act, slope
        self.weight = nn.Parameter(torch.ones(num_channels))
        self.bias = nn.Parameter(torch.zeros(num_channels))

    def forward(self, x, residual=None):
        return group_norm_act(x, self.num_groups, self.weight, self.bias, self.eps, self.act, self.slope, residual)


def dropout(x, p, rng, site=0, residual=None):
    """residual + dropout(x), goenv_dropout: an element is dropped with probability round(p * 65536) / 65536 and scaled
    by the inverse of what is kept; the mask is a function of (seed, step, site, place in memory).

    x: dense (contiguous or channels last), float32, bfloat16 or float16.  rng: int64 tensor [2] = (seed, step) on x's
    device; the kernel reads it, so a captured graph draws new masks when `step` is advanced between replays
    (``rng[1] += 1``, :meth:`DropoutState.advance`).  Advance it once per training step, after the backward pass: a
    backward pass whose rng has changed since its forward pass is refused by torch.  site: tells the layers of a step
    apart.  residual: of x's shape, type and strides.  Gradients for x and residual."""
    return _ops().dropout(x, p, rng, site, residual)


class DropoutState(nn.Module):
    """The (seed, step) of a network's dropout layers, as a buffer of it; layers take a site each.  Data-parallel ranks hold
    the same buffer: for masks of its own a rank adds rank * sites to its sites."""

    def __init__(self, seed=0):
        super().__init__()
        self.register_buffer("rng", torch.tensor([seed, 0], dtype=torch.int64))
        self.sites = 0

    def new_site(self):
        self.sites += 1
        return self.sites - 1

    def advance(self):
        """The next step's masks; once per training step, after its backward pass."""
        self.rng[1].add_(1)


def policy_logits(logits, legal=None, legal_bits=None, bias=None, history=None, history_len=None, repetition=1.0,
                  presence=0.0, frequency=0.0, temperature=1.0, out="logits", dtype=None):
    """Rows of logits under the game's rules, goenv_policy_logits: penalties for columns that stand in the row's
    history, a bias, a temperature and a mask, in this order; as "logits", "log_probs" or "probs".

    logits: [rows, cols], rows of any stride.  legal: uint8 or bool [rows, cols], 0 = forbidden (an environment's
    legal_out); legal_bits: int32 [rows, ceil(cols / 32)], bit v % 32 of word v // 32 = allowed; not both.  bias: [cols] or
    [rows, cols], float32 or the logits' type.  history: int32 or int64 [rows, h]; entries outside [0, cols), such as
    a pass, are skipped; history_len: int32 [rows], how many of a row's entries count (None: all).  repetition,
    presence, frequency, temperature: numbers, or float32 tensors [rows].  dtype: of the result, float32 or the logits'
    type (None: the logits' type).  Forbidden columns give -inf, or 0 as probabilities; so does a row with nothing left.
    Gradients for logits and bias: of the masks and histories that the call read (it copies them where gradients are wanted,
    so the environment may write the next position's into the same tensors before the backward pass)."""
    return _ops().policy_logits(logits, legal, legal_bits, bias, history, history_len, repetition, presence, frequency,
                                temperature, out, dtype)
