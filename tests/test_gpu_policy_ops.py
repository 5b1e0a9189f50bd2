"""GPU: the policy-network operators (elf_amd/policy_ops.py) against their definitions in 64 bits, within bounds that
policy_ops_ref.py derives from the roundings of a float32 computation."""
import pytest
import torch

import policy_ops_ref as ref
from policy_ops_ref import U, assert_within, wide

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def ops():
    from elf_amd import goenv, policy_ops
    goenv.load_library()
    assert torch.cuda.is_available()
    return policy_ops


@pytest.fixture(scope="module")
def error():
    from elf_amd import goenv
    return goenv.GoEnvError


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def normal(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g).to(dtype).cuda()


def image(g, n, c, spatial, dtype, scale=1.0, shift=0.0):
    """[n, c, *spatial], channels last."""
    return ((torch.randn(n, *spatial, c, generator=g) * scale + shift).to(dtype).cuda()).movedim(-1, 1)


# ---- group norm -------------------------------------------------------------------------------------------------
NORM = [
    # n, c, groups, positions, dtype, act, residual, type of weight and bias (None: none)
    (1, 1, 1, (1,), F32, "none", False, F32),
    (1, 8, 2, (), F32, "relu", True, F32),
    (1, 128, 8, (19, 19), BF16, "leaky_relu", True, F32),
    (3, 128, 8, (19, 19), BF16, "leaky_relu", True, BF16),
    (5, 128, 32, (19, 19), F16, "relu", False, F32),
    (9, 256, 32, (9, 9), F32, "silu", True, F32),
    (37, 120, 24, (13, 9), F32, "relu", False, F32),
    (2, 6, 3, (7,), F16, "silu", False, F16),
    (5, 33, 33, (5, 5), F32, "leaky_relu", True, None),
    (2, 40, 1, (17, 3), BF16, "none", True, F32),
    (2, 320, 32, (33, 31), BF16, "silu", False, F32),
    (3, 96, 4, (3, 5, 7), F32, "silu", True, F32),
    (2, 64, 4, (61, 67), F16, "silu", True, F32),
    (1, 32, 1, (80, 90), F32, "leaky_relu", False, F32),
    (1, 32, 1, (80, 90), BF16, "relu", True, F32),
    (1, 16, 8, (200, 201), F16, "silu", False, F32),
    (1, 7, 1, (150, 151), F32, "none", True, F32),
    (300, 24, 6, (2, 2), BF16, "leaky_relu", False, F32),
    (2, 5000, 1, (3,), BF16, "leaky_relu", True, F32),          # groups wider than a workgroup's vectors
    (2, 1025, 1, (5,), F32, "silu", False, F32),
    (2, 4096, 1, (7,), BF16, "silu", True, F32),                # ... or than their sums in LDS
    (3, 3000, 1, (9,), F16, "relu", False, F32),
    (130, 96, 32, (25, 25), F16, "relu", True, F32),
    (40, 15, 5, (23, 9), BF16, "silu", True, F32),
    (3, 240, 24, (50, 51), BF16, "leaky_relu", True, F32),
    (2, 128, 128, (40, 41), F32, "none", False, F32),
    (9000, 512, 1, (), BF16, "relu", True, F32),                # few positions: several samples a workgroup, one after the other
    (3000, 64, 8, (1,), F32, "silu", False, F32),
    (700, 120, 24, (2,), BF16, "silu", True, BF16),
    (33, 6, 6, (3, 3), F16, "relu", False, F32),
    (500, 960, 320, (2, 2), F32, "leaky_relu", True, F32),      # more groups than a workgroup has teams
    (70, 80, 2, (3,), BF16, "none", True, None),
    (40, 264, 1, (3,), F16, "silu", False, F16),
    (11, 528, 1, (2,), BF16, "leaky_relu", True, F32),          # a wave's lanes do not hold a position
]
ids = lambda v: str(v).replace("torch.", "").replace(" ", "")                             # noqa: E731


def norm_inputs(case, seed, shift=0.5):
    n, c, groups, spatial, dtype, act, residual, wt = case
    g = gen(seed)
    x = image(g, n, c, spatial, dtype, 1.5, shift)
    r = image(g, n, c, spatial, dtype) if residual else None
    w = None if wt is None else (1 + 0.3 * torch.randn(c, generator=g)).to(wt).cuda()
    b = None if wt is None else (0.3 * torch.randn(c, generator=g)).to(wt).cuda()
    return x, r, w, b, image(g, n, c, spatial, dtype)


def check_norm(ops, x, r, w, b, dy, groups, act, slope=0.1, eps=1e-5):
    leaves = {k: v.detach().requires_grad_(True) for k, v in dict(dx=x, dresidual=r, dweight=w, dbias=b).items() if v is not None}
    want = ref.group_norm_act(x, groups, w, b, eps, act, slope, r, dy)
    with torch.no_grad():
        assert_within(ops.group_norm_act(x, groups, w, b, eps, act, slope, r), want["y"], "y without gradients")
    y = ops.group_norm_act(leaves["dx"], groups, leaves.get("dweight"), leaves.get("dbias"), eps, act, slope, leaves.get("dresidual"))
    assert y.dtype == x.dtype and y.shape == x.shape
    assert_within(y, want["y"], "y")
    for (k, leaf), d in zip(leaves.items(), torch.autograd.grad(y, list(leaves.values()), dy)):
        assert d.dtype == leaf.dtype and d.shape == leaf.shape
        assert_within(d, want[k], k)


@pytest.mark.parametrize("case", NORM, ids=ids)
def test_group_norm(ops, case):
    x, r, w, b, dy = norm_inputs(case, 1)
    check_norm(ops, x, r, w, b, dy, case[2], case[5])


def test_group_norm_far_from_zero(ops):
    """A mean a thousand deviations away: sums of squares would lose the variance."""
    for dtype, spatial in ((F32, (19, 19)), (F32, (130, 140)), (F16, (19, 19))):
        case = (2, 32, 4, spatial, dtype, "leaky_relu", False, F32)
        x, r, w, b, dy = norm_inputs(case, 2, shift=1000.0)
        check_norm(ops, x, r, w, b, dy, 4, "leaky_relu")


def test_group_norm_of_views(ops):
    """Slices of channels, of samples, of positions; a gradient of another layout, an expanded one."""
    g = gen(3)
    big, bigr = image(g, 6, 96, (19, 11), BF16), image(g, 6, 104, (19, 11), BF16)
    for x, r in ((big[:, 8:72], bigr[:, 16:80]), (big[::2, :64], bigr[1:4, 3:67]), (big[:, 5:69, :7], None), (big[1:2, :64], bigr[3:4, :64])):
        w, b = normal(g, 64), normal(g, 64)
        check_norm(ops, x, r, w, b, normal(g, *x.shape, dtype=BF16), 8, "silu")           # dy: not channels last
        check_norm(ops, x, r, w, b, normal(g, 1, 64, 1, 1, dtype=BF16).expand(x.shape), 8, "leaky_relu")
    x = image(g, 3, 64, (9, 9), F32)
    nc = normal(g, 5, 64)[:, ::1]
    check_norm(ops, nc, None, None, None, normal(g, 5, 64), 4, "relu")
    check_norm(ops, x[:, :, ::1, 2:3], None, None, None, normal(g, 3, 64, 9, 1), 4, "relu")


def test_group_norm_unaligned(ops):
    """Arrays that start at any element."""
    g = gen(4)
    for dtype in (F32, BF16):
        for k in (1, 2, 4):
            def at(n, c, s):
                return normal(g, n * s * c + k, dtype=dtype)[k:].view(n, s, c).movedim(-1, 1)
            check_norm(ops, at(3, 64, 50), at(3, 64, 50), normal(g, 64 + k)[k:], normal(g, 64 + k)[k:], at(3, 64, 50), 8, "leaky_relu")
            check_norm(ops, at(7, 64, 3), at(7, 64, 3), None, None, at(7, 64, 3), 8, "silu")


def test_group_norm_empty(ops):
    for shape in ((0, 8, 3, 3), (2, 8, 0, 3)):
        x = torch.zeros(shape, device="cuda").to(memory_format=torch.channels_last).requires_grad_(True)
        w, b = torch.ones(8, device="cuda", requires_grad=True), torch.ones(8, device="cuda", requires_grad=True)
        y = ops.group_norm_act(x, 2, w, b)
        assert y.shape == shape
        dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.zeros_like(y))
        assert dx.shape == shape and not dw.any() and not db.any()


def test_group_norm_non_finite_samples_stay_apart(ops):
    x, r, w, b, dy = norm_inputs((4, 64, 8, (19, 19), BF16, "relu", True, F32), 5)
    clean = ops.group_norm_act(x, 8, w, b, residual=r, act="relu")
    bad = x.clone(memory_format=torch.preserve_format)
    bad[1, 3, 0, 0], bad[2, 60, 18, 18] = float("inf"), float("nan")
    y = ops.group_norm_act(bad, 8, w, b, residual=r, act="relu")
    same = torch.ones(4, 8, dtype=torch.bool)
    same[1, 0] = same[2, 7] = False
    for i in range(4):
        for k in range(8):
            part = y[i, 8 * k:8 * k + 8]
            assert torch.equal(part, clean[i, 8 * k:8 * k + 8]) if same[i, k] else bool(torch.isnan(part).all())


@pytest.mark.parametrize("case", [NORM[3], NORM[5], NORM[12], NORM[15], NORM[26], NORM[28]], ids=ids)
def test_group_norm_gives_equal_bits(ops, case):
    x, r, w, b, dy = norm_inputs(case, 6)
    for t in (x, r, w, b):
        if t is not None:
            t.requires_grad_(True)
    leaves = [t for t in (x, r, w, b) if t is not None]

    def once():
        y = ops.group_norm_act(x, case[2], w, b, act=case[5], residual=r)
        return (y,) + torch.autograd.grad(y, leaves, dy)
    first = once()
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(first, once()))


@pytest.mark.parametrize("spatial", [(19, 19), (70, 70)], ids=ids)
def test_group_norm_gradients_against_differences(ops, spatial):
    """Central differences of the kernel's own forward pass.  They are off by what they are off in 64 bits, and by the
    roundings of two outputs over 2 h."""
    x, r, w, b, dy = norm_inputs((2, 16, 4, spatial, F32, "silu", True, F32), 7)
    want = ref.group_norm_act(x, 4, w, b, 1e-5, "silu", 0.1, r, dy)
    inputs = dict(x=x, residual=r, weight=w, bias=b)
    leaves = {k: v.detach().clone(memory_format=torch.preserve_format).requires_grad_(True) for k, v in inputs.items()}
    y = ops.group_norm_act(leaves["x"], 4, leaves["weight"], leaves["bias"], act="silu", residual=leaves["residual"])
    got = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)))
    g, h = gen(8), 2.0 ** -6
    for k, v in inputs.items():
        way = torch.randn(v.shape, generator=g).cuda()
        sides, exact = [], []
        for s in (h, -h):
            moved = {**inputs, k: v + s * way}
            with torch.no_grad():
                z = ops.group_norm_act(moved["x"], 4, moved["weight"], moved["bias"], act="silu", residual=moved["residual"])
            e = ref.group_norm_act(moved["x"], 4, moved["weight"], moved["bias"], 1e-5, "silu", 0.1, moved["residual"])["y"]
            sides.append(float((wide(z) * wide(dy)).sum()))
            exact.append((float((e[0] * wide(dy)).sum()), float((e[1] * wide(dy).abs()).sum())))
        slope, slope64 = ((v[0] - v[1]) / (2 * h) for v in (sides, [exact[0][0], exact[1][0]]))
        formula, formula64 = (float((wide(d) * wide(way)).sum()) for d in (got[k], want["d" + k][0]))
        spare = float((want["d" + k][1] * wide(way).abs()).sum()) + (exact[0][1] + exact[1][1]) / (2 * h)
        assert abs(slope - formula) <= abs(slope64 - formula64) + spare, k


def test_group_norm_refusals(ops, error):
    x = image(gen(9), 2, 12, (5, 5), F32)
    w = torch.ones(12, device="cuda")
    for call, match in [
            (lambda: ops.group_norm_act(x.contiguous(), 4), "channels last"),
            (lambda: ops.group_norm_act(x[:, ::2], 2), "channels last"),
            (lambda: ops.group_norm_act(x[:, :, :, ::2], 2), "channels last"),
            (lambda: ops.group_norm_act(x.expand(2, 12, 5, 5)[:, :1].expand(2, 12, 5, 5), 2), "channels last"),
            (lambda: ops.group_norm_act(x.double(), 4), "float32"), (lambda: ops.group_norm_act(x[0, :, 0, 0], 4), "n, c"),
            (lambda: ops.group_norm_act(x, 5), "divides"), (lambda: ops.group_norm_act(x, 0), "divides"),
            (lambda: ops.group_norm_act(x, 4, w[:8]), "shape"), (lambda: ops.group_norm_act(x, 4, w.half()), "weight must be"),
            (lambda: ops.group_norm_act(x, 4, w.cpu()), "weight must be"), (lambda: ops.group_norm_act(x, 4, w, act="gelu"), "act"),
            (lambda: ops.group_norm_act(x, 4, w, eps=-1.0), "eps"), (lambda: ops.group_norm_act(x, 4, w, eps=float("nan")), "eps"),
            (lambda: ops.group_norm_act(x, 4, torch.ones(24, device="cuda")[::2]), "contiguous"),
            (lambda: ops.group_norm_act(x.bfloat16(), 4, w, w.bfloat16()), "one type"),
            (lambda: ops.group_norm_act(x, 4, residual=x.contiguous()), "channels last"),
            (lambda: ops.group_norm_act(x, 4, residual=x.half()), "residual must be"),
            (lambda: ops.group_norm_act(x, 4, residual=x[:1]), "residual must be"),
            (lambda: ops.group_norm_act(x, 4, act="leaky_relu", slope=float("inf")), "slope")]:
        with pytest.raises(error, match=match):
            call()


def test_group_norm_beyond_32_bit_offsets(ops):
    """The last samples of a tensor of 2.3 billion elements, forward and backward, against themselves alone (a sample's result
    does not depend on the others; the launch shapes differ, so within a rounding of the type)."""
    n, c = 50000, 128
    x = torch.randn(64, 19 * 19, c, device="cuda").to(BF16).repeat(n // 64 + 1, 1, 1)[:n]
    x[-3:] = torch.randn(3, 19 * 19, c, device="cuda").to(BF16)
    x = x.movedim(-1, 1).requires_grad_(True)
    y = ops.group_norm_act(x, 8, act="leaky_relu")
    (dx,) = torch.autograd.grad(y, x, x.detach())
    tail = x.detach()[-3:].clone(memory_format=torch.preserve_format)
    want = ref.group_norm_act(tail, 8, None, None, 1e-5, "leaky_relu", 0.1, None, tail)
    assert_within(y[-3:], want["y"])
    assert_within(dx[-3:], want["dx"])


# ---- dropout ----------------------------------------------------------------------------------------------------
def test_dropout_beyond_32_bit_offsets(ops):
    """The last elements of 2^32 + 13: the block counter's high word takes part from 2^35 elements on, offsets from 2^31."""
    n = (1 << 32) + 13
    x = torch.ones(n, dtype=BF16, device="cuda")
    y = ops.dropout(x, 0.5, rng_of(5, 6), 7)[-2061:].cpu()
    first = n - 2061
    assert first % 8 == 0
    kept = ref.keep_mask(2061, 5, 6, 7, 0.5, first // 8)
    assert torch.equal(y != 0, kept) and bool((y[kept] == 2).all())


def rng_of(seed, step):
    return torch.tensor([seed, step], dtype=torch.int64, device="cuda")


@pytest.mark.parametrize("n", [1, 2, 7, 8, 9, 63, 361, 722 * 5, 100003, 1 << 20], ids=ids)
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=ids)
@pytest.mark.parametrize("residual", [False, True], ids=["alone", "residual"])
def test_dropout(ops, n, dtype, residual):
    g = gen(n)
    x, dy = normal(g, n, dtype=dtype), normal(g, n, dtype=dtype)
    r = normal(g, n, dtype=dtype) if residual else None
    seed, step, site, p = 0x1234567890ABCDEF - n, n * 7, 5 + n, (0.1, 0.5, 0.37)[n % 3]
    xs, rs = x.clone().requires_grad_(True), r.clone().requires_grad_(True) if residual else None
    rng = rng_of(seed, step)
    y = ops.dropout(xs, p, rng, site, rs)
    want = ref.dropout(x, p, seed, step, site, r)
    assert_within(y, want, "y")
    with torch.no_grad():
        assert torch.equal(ops.dropout(x, p, rng, site, r), y.detach())
    kept = ref.keep_mask(n, seed, step, site, p)
    if not residual:                                 # the mask itself (randn gives no zero and no denormal)
        assert torch.equal(y.detach().cpu() != 0, kept)
    grads = torch.autograd.grad(y, (xs, rs) if residual else (xs,), dy)
    assert_within(grads[0], ref.dropout(dy, p, seed, step, site), "dx")
    assert torch.equal(grads[0].cpu() != 0, kept)
    if residual:
        assert torch.equal(grads[1], dy)


def test_dropout_ends_of_the_range(ops):
    g = gen(20)
    x = normal(g, 1000)
    x[3], x[5] = float("nan"), float("inf")
    r = normal(g, 1000)
    assert torch.equal(ops.dropout(x, 1.0, rng_of(1, 2)), torch.zeros_like(x))            # drops NaN too
    assert torch.equal(ops.dropout(x, 1.0, rng_of(1, 2), residual=r), r)
    y = ops.dropout(x, 0.0, rng_of(1, 2))
    assert torch.equal(torch.isnan(y), torch.isnan(x)) and torch.equal(y[6:], x[6:])
    assert ops.dropout(x[:0], 0.5, rng_of(1, 2)).numel() == 0
    kept = ref.keep_mask(1000, 77, 2, 0, 0.5)
    assert torch.equal(torch.isnan(ops.dropout(x, 0.5, rng_of(77, 2))).cpu(), kept & torch.isnan(x.cpu()))


def test_dropout_seeds_steps_and_sites(ops):
    x = torch.ones(4096, device="cuda")
    seen = []
    for seed, step, site in ((-1, 0, 0), (0, 0, 0), (1 << 62, 0, 0), (0, 1, 0), (0, (1 << 32) - 1, 0), (0, 0, 1), (0, 0, (1 << 32) - 1)):
        y = ops.dropout(x, 0.5, rng_of(seed, step), site)
        assert torch.equal(y.cpu() != 0, ref.keep_mask(4096, seed & ((1 << 64) - 1), step, site, 0.5))
        seen.append(y)
    for i in range(len(seen)):
        for k in range(i):
            assert 1700 < int((seen[i] != seen[k]).sum()) < 2400                          # 2,048 +- 11 deviations of 32


def test_dropout_layouts(ops, error):
    g = gen(21)
    x, r = image(g, 3, 24, (5, 7), BF16), image(g, 3, 24, (5, 7), BF16)
    xs = x.requires_grad_(True)
    y = ops.dropout(xs, 0.25, rng_of(9, 9), 1, r)
    assert y.stride() == x.stride()
    flat = lambda t: t.movedim(1, -1).reshape(-1)                                        # noqa: E731
    assert_within(flat(y.detach()), ref.dropout(flat(x), 0.25, 9, 9, 1, flat(r)))
    for dy in (normal(g, 3, 24, 5, 7, dtype=BF16), normal(g, 1, 1, 1, 1, dtype=BF16).expand(3, 24, 5, 7)):
        (dx,) = torch.autograd.grad(y, xs, dy, retain_graph=True)
        assert_within(flat(dx), ref.dropout(flat(dy), 0.25, 9, 9, 1))
    x = x.detach()
    for k in (1, 3):                                 # arrays that start at any element, of any length
        a, b = normal(g, 1003)[k:], normal(g, 1020)[9 - k:9 - k + 1003 - k]
        assert_within(ops.dropout(a, 0.5, rng_of(3, 4), 2, b), ref.dropout(a, 0.5, 3, 4, 2, b))
    for call, match in [
            (lambda: ops.dropout(x[:, ::2], 0.5, rng_of(0, 0)), "dense"), (lambda: ops.dropout(x[:, :1].expand(3, 4, 5, 7), 0.5, rng_of(0, 0)), "dense"),
            (lambda: ops.dropout(x, 1.5, rng_of(0, 0)), "p must be"), (lambda: ops.dropout(x, float("nan"), rng_of(0, 0)), "p must be"),
            (lambda: ops.dropout(x, True, rng_of(0, 0)), "p must be"),
            (lambda: ops.dropout(x, 0.5, rng_of(0, 0).int()), "rng must be"), (lambda: ops.dropout(x, 0.5, rng_of(0, 0).cpu()), "rng must be"),
            (lambda: ops.dropout(x, 0.5, rng_of(0, 0), -1), "site"), (lambda: ops.dropout(x, 0.5, rng_of(0, 0), 1 << 32), "site"),
            (lambda: ops.dropout(x, 0.5, torch.zeros(4, dtype=torch.int64, device="cuda")[::2]), "contiguous"),
            (lambda: ops.dropout(x, 0.5, rng_of(0, 0), residual=x.contiguous()), "strides"),
            (lambda: ops.dropout(x, 0.5, rng_of(0, 0), residual=x[:1]), "residual"), (lambda: ops.dropout(x.double(), 0.5, rng_of(0, 0)), "float32")]:
        with pytest.raises(error, match=match):
            call()


def test_dropout_refuses_a_backward_pass_after_the_next_step(ops):
    x = torch.ones(64, device="cuda", requires_grad=True)
    state = ops.DropoutState(5).cuda()
    y = ops.dropout(x, 0.5, state.rng, state.new_site())
    state.advance()
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()


# ---- policy logits ----------------------------------------------------------------------------------------------
def packed(legal):
    rows, cols = legal.shape
    bits = torch.zeros(rows, (cols + 31) // 32 * 32, dtype=torch.int64)
    bits[:, :cols] = legal.cpu()
    w = (bits.view(rows, -1, 32) << torch.arange(32)).sum(-1)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32).cuda()


LOGITS = [
    # rows, cols, dtype, out, result type, mask, bias, moves in the history, its type
    (1, 1, F32, "probs", None, "none", "none", 0, None),
    (1, 361, F32, "probs", F32, "bytes", "row", 8, torch.int32),
    (37, 361, BF16, "probs", F32, "bytes", "none", 8, torch.int64),
    (64, 361, F16, "log_probs", None, "bits", "shared", 3, torch.int32),
    (5, 362, F32, "log_probs", None, "bytes", "shared", 0, None),
    (3, 31, BF16, "logits", None, "bits", "row", 40, torch.int32),
    (130, 33, F32, "probs", None, "bits", "shared", 1, torch.int64),
    (7, 64, F16, "logits", F32, "none", "shared", 5, torch.int32),
    (4, 1000, BF16, "log_probs", F32, "bytes", "row", 100, torch.int32),
    (3, 4097, F32, "probs", None, "bits", "none", 600, torch.int32),
    (2, 16385, BF16, "logits", None, "bytes", "shared", 300, torch.int32),
    (2, 40000, F16, "log_probs", None, "bits", "shared", 513, torch.int64),
    (1, 131072, F16, "probs", F32, "bits", "none", 512, torch.int32),
    (3, 70001, F32, "log_probs", None, "none", "row", 0, None),
    (513, 17, F32, "logits", None, "bytes", "shared", 2, torch.int32),
    (9, 2, BF16, "probs", None, "bytes", "none", 0, None),
    (5, 3307, F32, "log_probs", None, "bits", "shared", 20, torch.int32),      # slices that are no power of two
    (6, 1537, BF16, "logits", None, "bytes", "row", 30, torch.int64),
    (3, 20666, F16, "probs", F32, "bits", "shared", 700, torch.int32),
    (2, 10004, F32, "probs", None, "none", "none", 0, None),
    (5, 9001, BF16, "log_probs", None, "bytes", "row", 300, torch.int32),
    (2, 12287, F32, "probs", None, "bits", "none", 40, torch.int64),
    (3, 12289, F16, "probs", F32, "bits", "none", 9, torch.int32),
]


def logit_inputs(case, seed):
    rows, cols, dtype, out, result, mask, bias, h, ht = case
    g = gen(seed)
    logits = (2 * torch.randn(rows, cols, generator=g)).to(dtype).cuda()
    legal = None
    if mask != "none":
        legal = torch.rand(rows, cols, generator=g) < 0.6
        if rows > 2:
            legal[rows // 2] = False                 # a row with nothing left
            legal[rows - 1] = False
            legal[rows - 1, cols // 2] = True        # and one with a single column
    kw = dict(repetition=(1 + torch.rand(rows, generator=g)).cuda(), presence=torch.rand(rows, generator=g).cuda(),
              frequency=torch.rand(rows, generator=g).cuda(), temperature=(0.5 + torch.rand(rows, generator=g)).cuda())
    if rows % 2:
        kw.update(repetition=1.25, temperature=0.75)
    if bias != "none":
        kw["bias"] = (0.5 * torch.randn(*((cols,) if bias == "shared" else (rows, cols)), generator=g)).to(F32 if rows != 7 else dtype).cuda()
    if h:
        kw["history"] = torch.randint(-2, cols + 2, (rows, h), generator=g).clamp_max(max(cols // 3, 1)).to(ht).cuda()
        if rows > 1:
            kw["history_len"] = torch.randint(-1, h + 3, (rows,), generator=g).to(torch.int32).cuda()   # clamped to 0 .. h
    dy = torch.randn(rows, cols, generator=g).to(result or dtype).cuda()
    return logits, legal, kw, dy


def check_logits(ops, case, logits, legal, kw, dy):
    out, result, mask = case[3], case[4], case[5]
    given = {} if legal is None else dict(legal=legal.to(torch.uint8).cuda()) if mask == "bytes" else dict(legal_bits=packed(legal))
    want = ref.policy_logits(logits, legal, out=out, dtype=result or logits.dtype, dy=dy, **kw)
    with torch.no_grad():
        assert_within(ops.policy_logits(logits, out=out, dtype=result, **given, **kw), want["y"], "y without gradients")
    leaves = dict(dlogits=logits.detach().requires_grad_(True))
    if "bias" in kw:
        leaves["dbias"] = kw["bias"].detach().requires_grad_(True)
        kw = {**kw, "bias": leaves["dbias"]}
    y = ops.policy_logits(leaves["dlogits"], out=out, dtype=result, **given, **kw)
    assert y.dtype == (result or logits.dtype) and y.is_contiguous()
    assert_within(y, want["y"], "y")
    for (k, leaf), d in zip(leaves.items(), torch.autograd.grad(y, list(leaves.values()), dy)):
        assert d.dtype == leaf.dtype and d.shape == leaf.shape
        assert_within(d, want[k], k)
    return y


@pytest.mark.parametrize("case", LOGITS, ids=ids)
def test_policy_logits(ops, case):
    check_logits(ops, case, *logit_inputs(case, 30))


def test_policy_logits_plain_softmax(ops):
    """No rule at all."""
    g = gen(31)
    for cols in (1, 361, 5000):
        for out in ("logits", "log_probs", "probs"):
            logits, dy = normal(g, 6, cols), normal(g, 6, cols)
            check_logits(ops, (6, cols, F32, out, None, "none"), logits, None, {}, dy)


def test_policy_logits_far_tails(ops):
    """Probabilities down to the smallest that float32 holds, and below."""
    g = gen(36)
    logits = -torch.linspace(0, 130, 2000)[torch.randperm(2000, generator=g)].view(4, 500).cuda()
    for out in ("probs", "log_probs"):
        case = (4, 500, F32, out, None, "none", "none", 0, None)
        check_logits(ops, case, logits, None, {}, normal(g, 4, 500))


def test_policy_logits_strides_and_types(ops):
    """Rows of any stride and start, masks of truth values, a gradient of another layout or expanded."""
    g = gen(32)
    wide_rows = normal(g, 9, 800)
    legal = torch.rand(9, 900, generator=g) < 0.5
    hist = torch.randint(-1, 361, (9, 20), generator=g).cuda()
    for k in (0, 1, 3):
        for dtype in (F32, BF16):
            x = wide_rows.to(dtype)[:, k:k + 361].detach().requires_grad_(True)
            m = legal.cuda()[:, 7 + k:7 + k + 361]
            h = hist[:, k:k + 9]
            want_of = lambda dy, out: ref.policy_logits(x, m, None, h, None, 1.5, 0.5, 0.25, 0.8, out, None, dy)  # noqa: E731
            for out in ("log_probs", "probs", "logits"):
                y = ops.policy_logits(x, legal=m, history=h, repetition=1.5, presence=0.5, frequency=0.25, temperature=0.8, out=out)
                for dy in (normal(g, 361, 9, dtype=dtype).t(), normal(g, 9, 1, dtype=dtype).expand(9, 361), normal(g, 9, 500, dtype=dtype)[:, 3:364]):
                    want = want_of(dy, out)
                    assert_within(y, want["y"])
                    assert_within(torch.autograd.grad(y, x, dy, retain_graph=True)[0], want["dlogits"])


def test_policy_logits_what_is_off_stays_off(ops):
    """Infinities, NaN and lowest values in forbidden columns, a bias of -inf as a mask, d_out of NaN there."""
    g = gen(33)
    for cols in (361, 9000):
        for out in ("logits", "log_probs", "probs"):
            logits, dy = normal(g, 6, cols), normal(g, 6, cols)
            legal = torch.rand(6, cols, generator=g) < 0.5
            legal[1], legal[2, 5:] = False, False
            bias = torch.zeros(6, cols)
            bias[3, ::2] = -float("inf")             # off by its bias
            bias[4] = -float("inf")
            bias[5, 1::2] = torch.finfo(F32).min     # not off: as low as a number can be
            clean = dict(bias=bias.cuda(), history=torch.randint(0, cols, (6, 4), generator=g).cuda(), repetition=2.0, presence=0.5)
            off = ~legal | (bias == -float("inf"))
            case = (6, cols, F32, out, None, "bytes")
            y = check_logits(ops, case, logits, legal, clean, torch.where(off.cuda(), 0.0, dy))
            assert torch.equal(y == (0 if out == "probs" else -float("inf")), off.cuda() | (y == (0 if out == "probs" else -float("inf"))))
            dirty = torch.where(legal.cuda(), logits, torch.tensor([float("nan"), float("inf"), -float("inf"), torch.finfo(F32).max, torch.finfo(F32).min] * cols,
                                                                  device="cuda")[:cols])
            bad_bias = torch.where(legal, bias, float("nan")).cuda()
            x = dirty.requires_grad_(True)
            z = ops.policy_logits(x, legal=legal.cuda(), out=out, **{**clean, "bias": bad_bias})
            assert torch.equal(z.detach(), y.detach())
            (dx,) = torch.autograd.grad(z, x, torch.where(off.cuda(), float("nan"), dy))
            x2 = logits.clone().requires_grad_(True)
            (dx2,) = torch.autograd.grad(ops.policy_logits(x2, legal=legal.cuda(), out=out, **clean), x2, torch.where(off.cuda(), 0.0, dy))
            assert torch.equal(dx, dx2) and not dx[off.cuda()].any()


def test_policy_logits_non_finite_rows_stay_apart(ops):
    g = gen(34)
    for cols in (361, 20000):
        logits = normal(g, 4, cols)
        clean = ops.policy_logits(logits, out="probs")
        logits[1, 7], logits[2, cols - 1] = float("nan"), float("inf")
        y = ops.policy_logits(logits, out="probs")
        assert torch.equal(y[0], clean[0]) and torch.equal(y[3], clean[3]) and bool(torch.isnan(y[1]).all()) and bool(torch.isnan(y[2, cols - 1]))


@pytest.mark.parametrize("case", [LOGITS[2], LOGITS[3], LOGITS[8], LOGITS[11]], ids=ids)
def test_policy_logits_gives_equal_bits(ops, case):
    logits, legal, kw, dy = logit_inputs(case, 35)
    given = dict(legal=legal.cuda()) if case[5] == "bytes" else dict(legal_bits=packed(legal))
    leaves = [logits.requires_grad_(True)] + ([kw["bias"].requires_grad_(True)] if "bias" in kw else [])

    def once():
        y = ops.policy_logits(logits, out=case[3], dtype=case[4], **given, **kw)
        return (y,) + torch.autograd.grad(y, leaves, dy)
    first = once()
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(first, once()))


@pytest.mark.parametrize("cols", [361, 9001])
@pytest.mark.parametrize("out", ["log_probs", "probs", "logits"])
def test_policy_logits_gradients_against_differences(ops, cols, out):
    """Central differences of the kernel's own forward pass; no logit or penalised logit near the kink at zero."""
    g = gen(36)
    logits = torch.randn(3, cols, generator=g)
    logits = torch.where(logits.abs() < 0.25, 0.5, logits).cuda()
    bias, dy = normal(g, cols), normal(g, 3, cols)
    legal = torch.rand(3, cols, generator=g) < 0.7
    dy = torch.where(legal.cuda(), dy, 0.0)
    kw = dict(history=torch.randint(0, cols, (3, 50), generator=g).cuda(), repetition=1.5, presence=0.25, frequency=0.5, temperature=0.8)
    want = ref.policy_logits(logits, legal, bias, out=out, dy=dy, **kw)
    x, b = logits.clone().requires_grad_(True), bias.clone().requires_grad_(True)
    y = ops.policy_logits(x, legal=legal.cuda(), bias=b, out=out, **kw)
    got = dict(zip(("logits", "bias"), torch.autograd.grad(y, (x, b), dy)))
    h = 2.0 ** -6
    live = lambda t: torch.where(legal, wide(t), 0.0)                                    # noqa: E731
    for k, v in (("logits", logits), ("bias", bias)):
        way = torch.rand(v.shape, generator=g).cuda() * 2 - 1                            # |h way| < 1/64: no sign changes
        sides, exact, spare = [], [], 0.0
        for s in (h, -h):
            moved = {"logits": logits, "bias": bias, k: v + s * way}
            sides.append(float((live(ops.policy_logits(moved["logits"], legal=legal.cuda(), bias=moved["bias"], out=out, **kw)) * wide(dy)).sum()))
            e = ref.policy_logits(moved["logits"], legal, moved["bias"], out=out, **kw)["y"]
            exact.append(float((live(e[0]) * wide(dy)).sum()))
            spare += float((e[1] * wide(dy).abs()).sum()) / (2 * h)
        slope, slope64 = ((p[0] - p[1]) / (2 * h) for p in (sides, exact))
        formula, formula64 = (float((wide(d) * wide(way)).sum()) for d in (got[k], want["d" + k][0]))
        spare += float((want["d" + k][1] * wide(way).abs()).sum())
        assert abs(slope - formula) <= abs(slope64 - formula64) + spare, k


def test_policy_logits_beyond_32_bit_offsets(ops):
    """The last rows of 2.3 billion logits, forward and backward."""
    rows, cols = 6_300_000, 361
    x = torch.randn(64, cols, device="cuda").to(BF16).repeat(rows // 64 + 1, 1)[:rows]
    x[-2:] = torch.randn(2, cols, device="cuda").to(BF16)
    legal = (torch.arange(cols, device="cuda") % 3 > 0).expand(rows, cols)
    x.requires_grad_(True)
    y = ops.policy_logits(x, legal=legal, out="log_probs")
    (dx,) = torch.autograd.grad(y, x, x.detach())
    tail = x.detach()[-2:]
    want = ref.policy_logits(tail, legal[-2:], out="log_probs", dy=tail)
    assert_within(y[-2:], want["y"])
    assert_within(dx[-2:], want["dlogits"])


def test_policy_logits_empty(ops):
    for shape in ((0, 361), (3, 0)):
        x, b = torch.zeros(shape, device="cuda", requires_grad=True), torch.zeros(shape[1], device="cuda", requires_grad=True)
        y = ops.policy_logits(x, bias=b, out="log_probs")
        dx, db = torch.autograd.grad(y, (x, b), torch.zeros_like(y))
        assert y.shape == shape and dx.shape == shape and not db.any()
    x = torch.randn(2, 5, device="cuda")
    assert torch.equal(ops.policy_logits(x, history=torch.zeros(2, 0, dtype=torch.int32, device="cuda"), repetition=2.0), x)


def test_policy_logits_refusals(ops, error):
    x = torch.randn(4, 40, device="cuda")
    m, w = torch.ones(4, 40, dtype=torch.uint8, device="cuda"), torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    h = torch.zeros(4, 6, dtype=torch.int32, device="cuda")
    for kw, match in [
            (dict(logits=x.double()), "float32"), (dict(logits=x[0]), "rows, cols"), (dict(logits=x.t()), "next to each other"),
            (dict(legal=m, legal_bits=w), "not both"), (dict(legal=m[:2]), "legal must be"), (dict(legal=m.float()), "legal must be"),
            (dict(legal=m.cpu()), "legal must be"), (dict(legal=m.t().contiguous().t()), "next to each other"),
            (dict(legal_bits=w[:, :1]), "legal_bits must be"), (dict(legal_bits=w.long()), "legal_bits must be"),
            (dict(bias=x[:, :39]), "bias must be"), (dict(bias=x[0, :39]), "bias must be"), (dict(bias=x.half()), "bias must be"),
            (dict(bias=x.t().contiguous().t()), "contiguous"), (dict(history=h[:3]), "history must be"), (dict(history=h.float()), "history must be"),
            (dict(history=h[0]), "history must be"), (dict(history=h.t().contiguous().t()), "next to each other"),
            (dict(history_len=h[:, 0].contiguous()), "without history"), (dict(history=h, history_len=h[:, 0].long()), "history_len must be"),
            (dict(history=h, history_len=h[:, 0]), "contiguous"), (dict(out="softmax"), "out must be"), (dict(dtype=torch.float16), "dtype must be"),
            (dict(temperature=0.0), "temperature"), (dict(temperature=-1), "temperature"), (dict(temperature=float("nan")), "temperature"),
            (dict(history=h, repetition=0.0), "repetition"), (dict(history=h, presence=float("inf")), "presence"),
            (dict(temperature=torch.ones(4, device="cuda", requires_grad=True)), "no gradient"), (dict(temperature=torch.ones(3, device="cuda")), "temperature must be"),
            (dict(temperature=torch.ones(4, device="cuda").double()), "temperature must be"), (dict(presence="1"), "must be a number")]:
        with pytest.raises(error, match=match):
            ops.policy_logits(**{"logits": x, **kw})
