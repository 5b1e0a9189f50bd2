"""The policy network's operators around its convolutions (libgoenv.so, include/goenv.h "Policy-network operators"):

* :func:`group_norm_act` -- group norm of a channels-last tensor, the residual sum and the activation of a block
* :func:`dropout`        -- dropout from a counter-based generator; the mask is never stored
* :func:`policy_logits`  -- penalties for repeated moves, biases, legal masks and a temperature on policy logits,
  as logits, log probabilities or the probabilities that ``GoEnv.sample_policy`` / ``topk_policy`` take

All of them take torch-ROCm tensors, run on torch's current stream of the tensors' device, allocate their outputs (and
nothing that outlives the call) through torch, and can be captured into a graph.  Gradients: once, through
``torch.autograd``.  There is no CPU fallback.
"""
import ctypes as C

import torch
import torch.nn as nn

from .goenv import ACTS, DTYPES, OUT_KINDS, GoEnvError, LogitRules, Norm, load_library


def _fail(*what):
    raise GoEnvError(what[0] % what[1:] if len(what) > 1 else what[0])


def _stream(device):
    return torch.cuda.current_stream(device).cuda_stream


def _check_rc(lib, rc):
    if rc != 0:
        raise GoEnvError(lib.goenv_last_error().decode())


def _is_float(t, name):
    if not torch.is_tensor(t) or t.device.type != "cuda":
        _fail("%s must be a tensor on the GPU", name)
    if t.dtype not in DTYPES:
        _fail("%s must be float32, bfloat16 or float16 (got %s)", name, t.dtype)


def _like(t, name, device, dtypes, shape):
    if not torch.is_tensor(t) or t.device != device or t.dtype not in dtypes or tuple(t.shape) != tuple(shape):
        _fail("%s must be a tensor of %s of shape %s on %s (got %s)", name, " or ".join(str(d) for d in dtypes), tuple(shape),
              device, "%s %s on %s" % (t.dtype, tuple(t.shape), t.device) if torch.is_tensor(t) else type(t).__name__)


def _wants_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# ---- group norm -------------------------------------------------------------------------------------------------
def _layout(t):
    """(sample stride, position stride) of a channels-last [n, c, *positions] tensor, None if it is not one."""
    shape, stride = t.shape, t.stride()
    if shape[1] != 1 and stride[1] != 1:
        return None
    position = want = 0
    for d in range(len(shape) - 1, 1, -1):
        if shape[d] == 1:
            continue
        if not position:
            position = stride[d]
        elif stride[d] != want:
            return None
        want = stride[d] * shape[d]
    return (stride[0] if shape[0] != 1 else 0), position


def _dense_like(t):
    """An empty tensor of t's shape and type, dense and channels last."""
    s = t.shape
    return torch.empty((s[0],) + tuple(s[2:]) + (s[1],), dtype=t.dtype, device=t.device).movedim(-1, 1)


def _channels_last(t):
    """t itself where its layout will do, else a dense channels-last copy."""
    at = _layout(t)
    if at is None:
        t = _dense_like(t).copy_(t)
        at = _layout(t)
    return t, at


def _norm_args(x, residual, weight, bias, groups, eps, act, slope, stats):
    shape = x.shape
    positions = 1
    for d in shape[2:]:
        positions *= d
    p = Norm()
    p.device, p.dtype, p.act = x.device.index, DTYPES[x.dtype], act
    p.n, p.positions, p.channels, p.groups = shape[0], positions, shape[1], groups
    p.eps, p.slope = eps, slope
    p.x = x.data_ptr()
    p.x_sample, p.x_position = _layout(x)
    if residual is not None:
        p.residual = residual.data_ptr()
        p.r_sample, p.r_position = _layout(residual)
    if weight is not None:
        p.weight, p.param_dtype = weight.data_ptr(), DTYPES[weight.dtype]
    if bias is not None:
        p.bias, p.param_dtype = bias.data_ptr(), DTYPES[bias.dtype]
    if stats is not None:
        p.stats = stats.data_ptr()
    return p


def _norm_workspace(lib, p, device, grad):
    need = lib.goenv_group_norm_workspace(p.n, p.positions, p.channels, p.groups, p.dtype, grad)
    if need <= 0:
        return None
    ws = torch.empty(need, dtype=torch.uint8, device=device)
    p.workspace, p.workspace_bytes = ws.data_ptr(), need
    return ws


def _norm_forward(x, residual, weight, bias, groups, eps, act, slope, stats):
    lib = load_library()
    y = _dense_like(x)
    p = _norm_args(x, residual, weight, bias, groups, eps, act, slope, stats)
    ws = _norm_workspace(lib, p, x.device, 0)  # noqa: F841 (held until the launch)
    _check_rc(lib, lib.goenv_group_norm_act(C.byref(p), y.data_ptr(), _stream(x.device)))
    return y


class _GroupNormAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, bias, groups, eps, act, slope):
        stats = torch.empty(x.shape[0], groups, 2, dtype=torch.float32, device=x.device)
        y = _norm_forward(x, residual, weight, bias, groups, eps, act, slope, stats)
        ctx.save_for_backward(x, residual, weight, bias, stats)
        ctx.how = groups, eps, act, slope
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, residual, weight, bias, stats = ctx.saved_tensors
        need = ctx.needs_input_grad
        dy, at = _channels_last(dy)
        lib = load_library()
        dx = _dense_like(x) if need[0] else None
        dr = _dense_like(x) if residual is not None and need[1] else None
        dw = torch.empty_like(weight) if weight is not None and need[2] else None
        db = torch.empty_like(bias) if bias is not None and need[3] else None
        p = _norm_args(x, residual, weight, bias, *ctx.how, stats)
        ws = _norm_workspace(lib, p, x.device, 1)  # noqa: F841
        _check_rc(lib, lib.goenv_group_norm_act_grad(
            C.byref(p), dy.data_ptr(), at[0], at[1], *(None if t is None else t.data_ptr() for t in (dx, dr, dw, db)),
            _stream(x.device)))
        return dx, dr, dw, db, None, None, None, None


def group_norm_act(x, num_groups, weight=None, bias=None, eps=1e-5, act="none", slope=0.1, residual=None):
    """act(group_norm(x) * weight + bias + residual), goenv_group_norm_act.

    x: [n, c, *positions], float32, bfloat16 or float16, channels last (``memory_format=torch.channels_last``, or any
    view whose channels lie next to each other: a slice of channels, of samples).  Statistics are taken per sample
    over the positions and the c / num_groups channels of a group, in float32.  weight, bias: [c], float32 or x's
    type.  residual: of x's shape and type, channels last.  act: "none", "relu", "leaky_relu" (with `slope`) or
    "silu".  The result is dense and channels last, of x's type.  Gradients for x, residual, weight and bias."""
    _is_float(x, "x")
    if x.dim() < 2:
        _fail("x must be [n, c, *positions] (got %s)", tuple(x.shape))
    if _layout(x) is None:
        _fail("x must be channels last (x.to(memory_format=torch.channels_last)); got shape %s, strides %s",
              tuple(x.shape), x.stride())
    c = x.shape[1]
    if not isinstance(num_groups, int) or num_groups <= 0 or c % num_groups:
        _fail("num_groups must be a positive integer that divides the %d channels (got %r)", c, num_groups)
    if act not in ACTS:
        _fail("act must be one of %s (got %r)", ", ".join(ACTS), act)
    if residual is not None:
        _like(residual, "residual", x.device, (x.dtype,), x.shape)
        if _layout(residual) is None:
            _fail("residual must be channels last, as x")
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is not None:
            _like(t, name, x.device, (torch.float32, x.dtype), (c,))
            if not t.is_contiguous():
                _fail("%s must be contiguous", name)
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        _fail("weight and bias must be of one type (got %s and %s)", weight.dtype, bias.dtype)
    args = (x, residual, weight, bias, num_groups, float(eps), ACTS[act], float(slope))
    if _wants_grad(x, residual, weight, bias):
        return _GroupNormAct.apply(*args)
    return _norm_forward(*args, None)


class GroupNormAct(nn.Module):
    """group_norm_act with a float32 weight and bias of its own; forward(x, residual=None)."""

    def __init__(self, num_groups, num_channels, eps=1e-5, act="none", slope=0.1):
        super().__init__()
        self.num_groups, self.eps, self.act, self.slope = num_groups, eps, act, slope
        self.weight = nn.Parameter(torch.ones(num_channels))
        self.bias = nn.Parameter(torch.zeros(num_channels))

    def forward(self, x, residual=None):
        return group_norm_act(x, self.num_groups, self.weight, self.bias, self.eps, self.act, self.slope, residual)


# ---- dropout ----------------------------------------------------------------------------------------------------
def _dense(t):
    """Whether t's elements fill its memory without gaps, in some order of the dimensions."""
    if t.is_contiguous():
        return True
    want = 1
    for stride, size in sorted((s, d) for s, d in zip(t.stride(), t.shape) if d != 1):
        if stride != want:
            return False
        want *= size
    return True


def _same_order(a, b):
    return all(x == y or d == 1 for x, y, d in zip(a.stride(), b.stride(), a.shape))


def _dropout_run(x, residual, p, rng, site):
    lib = load_library()
    y = torch.empty_strided(x.shape, x.stride(), dtype=x.dtype, device=x.device)
    _check_rc(lib, lib.goenv_dropout(x.device.index, DTYPES[x.dtype], x.numel(), x.data_ptr(),
                                     None if residual is None else residual.data_ptr(), y.data_ptr(), p, rng.data_ptr(),
                                     site, _stream(x.device)))
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, rng, site):
        ctx.save_for_backward(rng)
        ctx.how = p, site, x.stride()
        return _dropout_run(x, residual, p, rng, site)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        (rng,) = ctx.saved_tensors
        p, site, stride = ctx.how
        dx = None
        if ctx.needs_input_grad[0]:
            g = dy
            if g.stride() != stride:
                g = torch.empty_strided(dy.shape, stride, dtype=dy.dtype, device=dy.device).copy_(dy)
            dx = _dropout_run(g, None, p, rng, site)
        return dx, (dy if ctx.needs_input_grad[1] else None), None, None, None


def dropout(x, p, rng, site=0, residual=None):
    """residual + dropout(x), goenv_dropout: an element is dropped with probability round(p * 65536) / 65536 and scaled
    by the inverse of what is kept; the mask is a function of (seed, step, site, place in memory).

    x: dense (contiguous or channels last), float32, bfloat16 or float16.  rng: int64 tensor [2] = (seed, step) on x's
    device; the kernel reads it, so a captured graph draws new masks when `step` is advanced between replays
    (``rng[1] += 1``, :meth:`DropoutState.advance`).  Advance it once per training step, after the backward pass: a
    backward pass whose rng has changed since its forward pass is refused by torch.  site: tells the layers of a step
    apart.  residual: of x's shape, type and strides.  Gradients for x and residual."""
    _is_float(x, "x")
    if not _dense(x):
        _fail("x must be dense (contiguous or channels last); got shape %s, strides %s", tuple(x.shape), x.stride())
    if isinstance(p, bool) or not isinstance(p, (int, float)) or not 0.0 <= p <= 1.0:
        _fail("p must be a number from 0 to 1 (got %r)", p)
    if not isinstance(site, int) or not 0 <= site < 1 << 32:
        _fail("site must be an integer from 0 to 2^32 - 1 (got %r)", site)
    _like(rng, "rng", x.device, (torch.int64,), (2,))
    if not rng.is_contiguous():
        _fail("rng must be contiguous")
    if residual is not None:
        _like(residual, "residual", x.device, (x.dtype,), x.shape)
        if not _same_order(x, residual):
            _fail("residual must have x's strides (got %s and %s)", residual.stride(), x.stride())
    if _wants_grad(x, residual):
        return _Dropout.apply(x, residual, float(p), rng, site)
    return _dropout_run(x, residual, float(p), rng, site)


class DropoutState(nn.Module):
    """The (seed, step) of a network's dropout layers, as a buffer of it; layers take a site each."""

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


# ---- policy logits ----------------------------------------------------------------------------------------------
_PER_ROW = ("repetition", "presence", "frequency", "temperature")


def _logit_args(logits, legal, legal_bits, bias, history, history_len, params, kind, dtype, stats):
    p = LogitRules()
    p.device, p.dtype, p.out_dtype, p.out_kind = logits.device.index, DTYPES[logits.dtype], DTYPES[dtype], kind
    p.rows, p.cols = logits.shape
    p.logits, p.logits_row = logits.data_ptr(), logits.stride(0)
    if legal is not None:
        p.legal, p.legal_row = legal.data_ptr(), legal.stride(0)
    if legal_bits is not None:
        p.legal_bits, p.bits_row = legal_bits.data_ptr(), legal_bits.stride(0)
    if bias is not None:
        p.bias, p.bias_dtype, p.bias_row = bias.data_ptr(), DTYPES[bias.dtype], 0 if bias.dim() == 1 else bias.shape[1]
    if history is not None:
        p.history, p.history_row, p.history_max = history.data_ptr(), history.stride(0), history.shape[1]
        p.history_i64 = history.dtype == torch.int64
        if history_len is not None:
            p.history_len = history_len.data_ptr()
    p.repetition, p.presence, p.frequency, p.temperature = 1.0, 0.0, 0.0, 1.0
    for name, v in zip(_PER_ROW, params):
        if torch.is_tensor(v):
            setattr(p, "row_" + name, v.data_ptr())
        else:
            setattr(p, name, v)
    if stats is not None:
        p.stats = stats.data_ptr()
    return p


def _logit_workspace(lib, p, device, shared, grad):
    need = lib.goenv_policy_logits_workspace(p.rows, p.cols, p.out_kind, shared, grad)
    if need <= 0:
        return None
    ws = torch.empty(need, dtype=torch.uint8, device=device)
    p.workspace, p.workspace_bytes = ws.data_ptr(), need
    return ws


def _logits_forward(logits, legal, legal_bits, bias, history, history_len, params, kind, dtype, stats):
    lib = load_library()
    out = torch.empty(logits.shape, dtype=dtype, device=logits.device)
    p = _logit_args(logits, legal, legal_bits, bias, history, history_len, params, kind, dtype, stats)
    ws = _logit_workspace(lib, p, logits.device, bias is not None and bias.dim() == 1, 0)  # noqa: F841
    _check_rc(lib, lib.goenv_policy_logits(C.byref(p), out.data_ptr(), _stream(logits.device)))
    return out


class _PolicyLogits(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, bias, legal, legal_bits, history, history_len, params, kind, dtype, *row_params):
        stats = None
        if kind != OUT_KINDS["logits"]:
            stats = torch.empty(logits.shape[0], 2, dtype=torch.float32, device=logits.device)
        out = _logits_forward(logits, legal, legal_bits, bias, history, history_len, params, kind, dtype, stats)
        ctx.save_for_backward(logits, bias, legal, legal_bits, history, history_len, stats, *row_params)
        ctx.how = tuple(None if torch.is_tensor(v) else v for v in params), kind, dtype
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        logits, bias, legal, legal_bits, history, history_len, stats, *row_params = ctx.saved_tensors
        scalars, kind, dtype = ctx.how
        rows = iter(row_params)
        params = tuple(next(rows) if v is None else v for v in scalars)
        if dy.stride(1) != 1 and dy.shape[1] != 1:
            dy = dy.contiguous()
        lib = load_library()
        dl = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device) if ctx.needs_input_grad[0] else None
        db = torch.empty(bias.shape, dtype=bias.dtype, device=bias.device) if ctx.needs_input_grad[1] else None
        p = _logit_args(logits, legal, legal_bits, bias, history, history_len, params, kind, dtype, stats)
        ws = _logit_workspace(lib, p, logits.device, bias is not None and bias.dim() == 1, 1)  # noqa: F841
        _check_rc(lib, lib.goenv_policy_logits_grad(C.byref(p), dy.data_ptr(), dy.stride(0),
                                                    None if dl is None else dl.data_ptr(), None if db is None else db.data_ptr(),
                                                    _stream(logits.device)))
        return (dl, db) + (None,) * (7 + len(row_params))


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
    Gradients for logits and bias."""
    _is_float(logits, "logits")
    dev = logits.device
    if logits.dim() != 2:
        _fail("logits must be [rows, cols] (got %s)", tuple(logits.shape))
    rows, cols = logits.shape
    if logits.stride(1) != 1 and cols != 1:
        _fail("the columns of logits must lie next to each other (got strides %s)", logits.stride())
    if legal is not None:
        if legal_bits is not None:
            _fail("legal or legal_bits, not both")
        _like(legal, "legal", dev, (torch.uint8, torch.bool), (rows, cols))
        if legal.stride(1) != 1 and cols != 1:
            _fail("the columns of legal must lie next to each other")
    if legal_bits is not None:
        words = (cols + 31) // 32
        _like(legal_bits, "legal_bits", dev, (torch.int32,), (rows, words))
        if legal_bits.stride(1) != 1 and words != 1:
            _fail("the words of a row of legal_bits must lie next to each other")
    if bias is not None:
        _like(bias, "bias", dev, (torch.float32, logits.dtype), (cols,) if torch.is_tensor(bias) and bias.dim() == 1 else (rows, cols))
        if not bias.is_contiguous():
            _fail("bias must be contiguous")
    if history is not None:
        if not torch.is_tensor(history) or history.dim() != 2:
            _fail("history must be a tensor [rows, moves]")
        _like(history, "history", dev, (torch.int32, torch.int64), (rows, history.shape[1]))
        if history.stride(1) != 1 and history.shape[1] != 1:
            _fail("the entries of a row of history must lie next to each other")
    if history_len is not None:
        if history is None:
            _fail("history_len without history")
        _like(history_len, "history_len", dev, (torch.int32,), (rows,))
        if not history_len.is_contiguous():
            _fail("history_len must be contiguous")
    if out not in OUT_KINDS:
        _fail("out must be one of %s (got %r)", ", ".join(OUT_KINDS), out)
    if dtype is None:
        dtype = logits.dtype
    elif dtype not in (torch.float32, logits.dtype):
        _fail("dtype must be float32 or the logits' type (got %s)", dtype)
    params, row_params = [], []
    for name, v in zip(_PER_ROW, (repetition, presence, frequency, temperature)):
        if torch.is_tensor(v):
            _like(v, name, dev, (torch.float32,), (rows,))
            if not v.is_contiguous():
                _fail("%s must be contiguous", name)
            if v.requires_grad:
                _fail("%s has no gradient (detach it)", name)
            row_params.append(v)
        elif isinstance(v, bool) or not isinstance(v, (int, float)):
            _fail("%s must be a number or a float32 tensor [rows]", name)
        else:
            v = float(v)
        params.append(v)
    if _wants_grad(logits, bias):
        return _PolicyLogits.apply(logits, bias, legal, legal_bits, history, history_len, tuple(params), OUT_KINDS[out], dtype,
                                   *row_params)
    return _logits_forward(logits, legal, legal_bits, bias, history, history_len, params, OUT_KINDS[out], dtype, None)
