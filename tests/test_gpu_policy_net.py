"""GPU: the policy-network operators as they are used together -- a chain with its gradients, inside the policy/value net and its
training and selfplay commands, between the environment's masks and its sampler, in captured graphs, on several
streams and from several threads."""
import math
import os
import subprocess
import sys
import threading

import numpy as np
import pytest
import torch
import torch.nn.functional as F

import policy_ops_ref as ref
from common import ROOT
from oracle.pyoracle import OracleBoard

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    from elf_amd import goenv, policy_ops
    goenv.load_library()
    assert torch.cuda.is_available()
    return policy_ops


def chain_inputs(seed, n=6, c=32, dtype=torch.float32):
    g = torch.Generator()
    g.manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)                                          # noqa: E731
    t = dict(x=r(n, 19, 19, c).permute(0, 3, 1, 2), s=r(n, 19, 19, c).permute(0, 3, 1, 2), w1=1 + 0.2 * r(c), b1=0.2 * r(c), w2=1 + 0.2 * r(c),
             b2=0.2 * r(c), head=r(361, c) / c ** 0.5, bias=0.3 * r(361))
    t = {k: v.to(dtype) if k in ("x", "s", "head") else v for k, v in t.items()}
    legal = torch.rand(n, 361, generator=g) < 0.7
    legal[:, 0] = True
    return t, legal, torch.randint(0, 361, (n,), generator=g)


def chain(ops, t, legal, target, rng):
    """norm + sum + activation, dropout + sum, norm + activation, a head, log probabilities over the legal moves, a loss."""
    y = ops.group_norm_act(t["x"], 8, t["w1"], t["b1"], act="silu", residual=t["s"])
    y = ops.dropout(y, 0.25, rng, site=2, residual=t["s"])
    y = ops.group_norm_act(y, 4, t["w2"], t["b2"], act="silu")
    logits = y.mean((2, 3)).to(t["head"].dtype) @ t["head"].t()
    logp = ops.policy_logits(logits, legal=legal, bias=t["bias"], temperature=0.8, out="log_probs", dtype=torch.float32)
    logp = torch.where(legal, logp, 0.0)
    return -logp.gather(1, target[:, None]).mean() - 0.01 * logp.mean()


def chain64(t, legal, target, seed, step):
    n, c = t["x"].shape[:2]
    y = F.silu(F.group_norm(t["x"], 8, t["w1"], t["b1"], 1e-5) + t["s"])
    keep = ref.keep_mask(y.numel(), seed, step, 2, 0.25).view(n, 19, 19, c).permute(0, 3, 1, 2)
    y = torch.where(keep, y * (65536 / (65536 - ref.threshold(0.25))), 0.0) + t["s"]
    y = F.silu(F.group_norm(y, 4, t["w2"], t["b2"], 1e-5))
    z = (y.mean((2, 3)) @ t["head"].t() + t["bias"]) / 0.8
    logp = torch.log_softmax(torch.where(legal, z, -math.inf), 1)
    logp = torch.where(legal, logp, 0.0)
    return -logp.gather(1, target[:, None]).mean() - 0.01 * logp.mean()


def test_a_chain_of_all_three_and_its_gradients(ops):
    """Every function of the chain is smooth.  Ten stages (five forward, five back) of some 32 roundings each, and
    an amplification of at most 16 in all between relative errors: 10 * 32 * 16 * 2^-24 = 3e-4."""
    t, legal, target = chain_inputs(1)
    seed, step = 11, 3
    leaves = {k: v.cuda().requires_grad_(True) for k, v in t.items()}
    loss = chain(ops, leaves, legal.cuda(), target.cuda(), torch.tensor([seed, step], device="cuda"))
    grads = torch.autograd.grad(loss, list(leaves.values()))
    exact = {k: v.double().requires_grad_(True) for k, v in t.items()}
    loss64 = chain64(exact, legal, target, seed, step)
    grads64 = torch.autograd.grad(loss64, list(exact.values()))
    assert abs(float(loss.detach()) - float(loss64.detach())) <= 3e-4 * abs(float(loss64.detach()))
    for k, g, e in zip(t, grads, grads64):
        assert float((g.cpu().double() - e).norm()) <= 3e-4 * float(e.norm()), k


def test_a_training_step_in_a_captured_graph(ops):
    """Forward and backward of the chain, replayed with eager work between the replays, the dropout step advanced for each:
    every replay equals the eager result bit for bit.  The graph has leaves of its own."""
    t, legal, target = chain_inputs(2, dtype=BF16)
    legal, target = legal.cuda(), target.cuda()
    eager = {k: v.cuda().requires_grad_(True) for k, v in t.items()}
    static = {k: v.detach().clone(memory_format=torch.preserve_format).requires_grad_(True) for k, v in eager.items()}
    rng, rng_eager = torch.tensor([4, 0], device="cuda"), torch.tensor([4, 0], device="cuda")

    def step(leaves, state):
        loss = chain(ops, leaves, legal, target, state)
        return (loss.detach(),) + torch.autograd.grad(loss, list(leaves.values()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(static, rng)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static, rng)
    before = None
    for i in range(5):
        for state in (rng, rng_eager):
            state[1] = i
        graph.replay()
        want = step(eager, rng_eager)
        torch.cuda.synchronize()
        for k, (a, b) in enumerate(zip(out, want)):
            assert torch.equal(a, b), (i, k)
        assert before is None or not torch.equal(before, out[1])                         # another step, another mask
        before = out[1].clone()


def test_a_capture_refuses_leaves_of_a_living_eager_graph(ops):
    """The forward call is refused, before torch's engine would tie the default stream to the capture.  Without gradients, after
    the eager graph's end, or with a graph made on another stream that is not the default one, it is captured."""
    from elf_amd.goenv import GoEnvError
    w = torch.ones(8, device="cuda", requires_grad=True)
    x, l = torch.randn(2, 9, 8, device="cuda").transpose(1, 2), torch.randn(2, 8, device="cuda")
    rng = torch.tensor([1, 0], device="cuda")
    calls = [lambda: ops.group_norm_act(x, 2, w), lambda: ops.policy_logits(l, bias=w), lambda: ops.dropout(w, 0.5, rng)]
    want = [run() for run in calls]                                                      # three eager graphs of the leaf
    grads = [torch.autograd.grad(y.sum(), w, retain_graph=True)[0] for y in want]
    torch.cuda.synchronize()
    for run in calls:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            with torch.no_grad():
                out = run()                                                              # (so that the graph is not empty)
            with pytest.raises(GoEnvError, match="outside the capture"):
                run()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.isfinite(out).all()
    want = [y.detach() for y in want]
    for run, y, gw in zip(calls, want, grads):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
            got = torch.autograd.grad(out, w, torch.ones_like(out))[0]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, y) and torch.equal(got, gw)
        del out, got


def test_two_graphs_side_by_side(ops):
    """Long axes and long rows use workspaces; two captured graphs replayed at the same time on two streams have one each."""
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    made = []
    for i in range(2):
        x = torch.randn(1, 100, 100, 64, device="cuda", generator=g).permute(0, 3, 1, 2)
        l = torch.randn(2, 60000, device="cuda", generator=g)
        run = lambda x=x, l=l: (ops.group_norm_act(x, 8, act="silu"), ops.policy_logits(l, out="probs"))  # noqa: E731
        want = run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        made.append((graph, out, want, torch.cuda.Stream(), x, l))         # (a graph does not keep its inputs)
    for _ in range(20):
        for graph, _, _, stream, _, _ in made:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, out, want, *_ in made:
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_streams_and_threads(ops):
    """Four threads, a stream each, many calls at once, gradients among them."""
    t, legal, target = chain_inputs(3)
    legal, target = legal.cuda(), target.cuda()
    base = {k: v.cuda() for k, v in t.items()}

    def once():
        leaves = {k: v.detach().clone(memory_format=torch.preserve_format).requires_grad_(True) for k, v in base.items()}
        loss = chain(ops, leaves, legal, target, torch.tensor([4, 9], device="cuda"))
        return torch.autograd.grad(loss, list(leaves.values()))
    want = once()
    torch.cuda.synchronize()
    wrong, failed = [], []

    def work():
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(10):
                    got = once()
                    stream.synchronize()
                    wrong.extend(k for k, a, b in zip(t, got, want) if not torch.equal(a, b))
        except Exception as e:                       # noqa: BLE001
            failed.append(e)
    threads = [threading.Thread(target=work) for _ in range(4)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not failed and not wrong


def test_gradients_are_differentiable_once(ops):
    t, legal, target = chain_inputs(4, n=1)
    leaves = {k: v.cuda().requires_grad_(True) for k, v in t.items()}
    rng = torch.tensor([1, 1], device="cuda")
    for y, x in ((ops.group_norm_act(leaves["x"], 8, act="silu"), leaves["x"]), (ops.dropout(leaves["x"], 0.5, rng), leaves["x"]),
                 (ops.policy_logits(leaves["head"].t(), out="probs") if leaves["head"].t().stride(1) == 1 else
                  ops.policy_logits(leaves["head"], out="probs"), leaves["head"])):
        (d,) = torch.autograd.grad((y * y).sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="once"):
            torch.autograd.grad(d.sum(), x)


def test_between_the_environment_and_its_sampler(ops):
    """The environment's legal masks -> policy_logits -> sample_policy and topk_policy: what the sampler draws is what the oracle
    draws from the same pi, the forbidden points weigh nothing."""
    from elf_amd import goenv
    boards, seed = 48, 21
    env = goenv.GoEnv(boards, seed=seed, max_ply=722)
    env.ply_repeat(60, goenv.F_RANDOM_POLICY)
    legal, feat = env.new(torch.uint8, 361), env.new(torch.float32, 25, 19, 19)
    env.features(feat, legal_out=legal)
    past = torch.randint(-1, 361, (boards, 6), dtype=torch.int32, device=env.device)
    logits = torch.randn(boards, 361, device=env.device)
    kw = dict(legal=legal, history=past, repetition=1.5, presence=0.5, temperature=0.7, out="probs", dtype=torch.float32)
    pi = ops.policy_logits(logits, **kw)
    want = ref.policy_logits(logits, legal.bool(), history=past, repetition=1.5, presence=0.5, temperature=0.7, out="probs", dtype=torch.float32)
    ref.assert_within(pi, want["y"])
    assert not pi[legal == 0].any()
    acts = torch.zeros(boards, dtype=torch.int64, device=env.device)
    env.sample_policy(pi, acts)
    top, weights = env.new(torch.int32, 5), env.new(torch.float32, 5)
    env.topk_policy(pi, 5, top, weights)
    st = {k: v.cpu().numpy() for k, v in env.get_state().items()}
    pi_h, acts, top = pi.cpu().numpy(), acts.cpu().tolist(), top.cpu().numpy()
    for b in range(boards):
        o = OracleBoard()
        o.set_state(st["color"][b], st["last_placed"][b], st["scalars"][b])
        assert acts[b] == o.sample_policy(seed, b, 0, pi_h[b], 0)
        assert np.allclose(pi_h[b][top[b]], np.sort(pi_h[b])[::-1][:5], rtol=0, atol=0)
    env.close()


@pytest.mark.parametrize("dtype", [torch.float32, BF16], ids=["float32", "bfloat16"])
def test_the_net_with_group_norm_and_dropout(ops, dtype):
    """It trains a step (every parameter gets a finite gradient), a new step has new masks, evaluation has none; its policy over a
    legal mask sums to 1 over the legal points."""
    from elf_amd.df_model import PolicyValueNet
    torch.manual_seed(0)
    net = PolicyValueNet(dim=32, num_block=2, norm="group", groups=8, dropout=0.2).cuda().to(dtype).to(memory_format=torch.channels_last).train()
    s = torch.randn(5, 25, 19, 19, device="cuda")
    legal = (torch.rand(5, 361, device="cuda") < 0.5).to(torch.uint8)
    legal[4] = 0
    out = net(s)
    ((out["pi"].float() * torch.randn(5, 361, device="cuda")).sum() + out["V"].float().sum()).backward()
    assert all(p.grad is not None and bool(torch.isfinite(p.grad).all()) for p in net.parameters())
    assert torch.equal(net(s)["pi"], out["pi"])                                          # the same step, the same masks
    net.next_step()
    assert not torch.equal(net(s)["pi"], out["pi"])
    net.eval()
    with torch.no_grad():
        one = net(s, legal, 0.8)
        net.next_step()
        assert torch.equal(net(s, legal, 0.8)["pi"], one["pi"])
    assert one["pi"].dtype == torch.float32 and not one["pi"][legal == 0].any()
    with torch.no_grad():                                                                # a temperature per position
        assert torch.equal(net(s, temperature=torch.full((5,), 0.8, device="cuda"))["pi"], net(s, temperature=0.8)["pi"])
    sums = one["pi"].double().sum(1).cpu()
    # 361 probabilities of half a step each, the sum they were divided by off by (24 + 64) roundings
    assert float((sums[:4] - 1).abs().max()) <= (361 + 88) * 2.0 ** -24 and float(sums[4]) == 0


@pytest.mark.parametrize("cmd", [
    ["tools/df_train_gpu.py", "--num_games", "16", "--batchsize", "16", "--iters", "2", "--num_layer", "3", "--dim", "32", "--groups", "8",
     "--dropout", "0.1", "--fused_loss", "--bf16"],
    ["tools/df_selfplay_gpu.py", "--num_games", "16", "--batchsize", "16", "--iters", "3", "--num_block", "1", "--dim", "32", "--groups", "8",
     "--mask_policy", "--temperature", "0.8", "--bf16"]], ids=["train", "selfplay"])
def test_the_commands_that_use_them(cmd):
    out = subprocess.run([sys.executable, "-u", os.path.join(ROOT, cmd[0])] + cmd[1:], cwd=ROOT, capture_output=True, text=True, timeout=100)
    assert out.returncode == 0 and ("cfg3 train" in out.stdout or "cfg5" in out.stdout), out.stdout[-2000:] + out.stderr[-2000:]


def test_views_that_negate(ops):
    """A view may say that its memory holds the values with the other sign (the imaginary part of a conjugate): arguments,
    rules and gradients count with their values."""
    g = torch.Generator(device="cuda")
    g.manual_seed(8)
    randn = lambda *s: torch.randn(*s, device="cuda", generator=g)                       # noqa: E731

    def other(v):
        v = torch._neg_view(-v)
        assert v.is_neg()
        return v
    assert torch.complex(randn(3), randn(3)).conj().imag.is_neg()
    rng = torch.tensor([3, 0], device="cuda")
    x, r = (randn(3, 5, 8).transpose(1, 2) for _ in range(2))
    w, b, l, t, past = randn(8), randn(8), randn(4, 9), randn(4).abs() + 0.5, torch.randint(0, 9, (4, 3), device="cuda", generator=g)

    def same(run, *args):
        for got, want in zip(run(*[other(a) for a in args]), run(*args)):
            assert torch.equal(got, want)
    same(lambda x, r, w, b: (ops.group_norm_act(x, 2, w, b, act="silu", residual=r),), x, r, w, b)
    same(lambda x, r, rng: (ops.dropout(x, 0.5, rng, residual=r),), x, r, rng)
    same(lambda l, b, t, past: (ops.policy_logits(l, bias=b, history=past, temperature=t, presence=t, out="probs"),), l, randn(9), t, past)
    leaves = [v.detach().clone(memory_format=torch.preserve_format).requires_grad_(True) for v in (x, w, l)]
    same(lambda dy: torch.autograd.grad(ops.group_norm_act(leaves[0], 2, leaves[1], act="silu"), leaves[:2], dy), r)
    same(lambda dy: torch.autograd.grad(ops.dropout(leaves[0], 0.5, rng), leaves[0], dy), r)
    same(lambda dy: torch.autograd.grad(ops.policy_logits(leaves[2], out="log_probs"), leaves[2], dy), randn(4, 9))
