"""CPU: the policy-network operators' refusals, structures and generator (elf_amd/policy_ops.py, include/goenv.h), and the
64-bit definitions that the GPU tests hold the kernels to, against differences and known answers."""
import ctypes as C
import os
import subprocess

import pytest
import torch

import policy_ops_ref as ref
from common import ROOT


@pytest.fixture(scope="module")
def lib():
    from elf_amd import goenv
    return goenv.load_library()


def test_structures_match_the_header(tmp_path):
    from elf_amd import goenv
    src = tmp_path / "layout.c"
    lines = ["#include <stdio.h>", '#include "goenv.h"', "int main(void) {"]
    want = []
    for name, cls in (("goenv_norm", goenv.Norm), ("goenv_logit_rules", goenv.LogitRules)):
        lines.append('printf("%%zu\\n", sizeof(%s));' % name)
        want.append(C.sizeof(cls))
        for field, _ in cls._fields_:
            lines.append('printf("%%zu\\n", offsetof(%s, %s));' % (name, field))
            want.append(getattr(cls, field).offset)
    src.write_text("\n".join(lines + ["return 0; }"]))
    exe = str(tmp_path / "layout")
    subprocess.check_call(["gcc", "-I" + os.path.join(ROOT, "include"), str(src), "-o", exe])
    assert [int(v) for v in subprocess.check_output([exe]).split()] == want


# published known answers of Philox4x32-10 (counter, key, result)
@pytest.mark.parametrize("counter,key,want", [
    ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
    ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
    ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
     (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))])
def test_generator_known_answers(counter, key, want):
    assert tuple(int(v) for v in ref.philox(counter, key)) == want


def test_generator_is_fair():
    n = 1 << 20
    for p in (0.1, 0.5, 0.9):
        kept = float(ref.keep_mask(n, 12345, 6, 7, p).double().mean())
        q = 1 - ref.threshold(p) / 65536
        assert abs(kept - q) < 6 * (q * (1 - q) / n) ** 0.5          # six standard deviations


def test_definitions_against_differences():
    """The formulas of the gradients against central differences of the 64-bit definitions themselves."""
    g = torch.Generator().manual_seed(3)
    d = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)                     # noqa: E731
    h = 1e-5

    def agree(f, inputs, names, dy, **kw):
        got = f(**inputs, dy=dy, **kw)
        for name, key in names.items():
            way = d(*inputs[key].shape)
            at = [(f(**{**inputs, key: inputs[key] + s * way}, **kw)["y"][0] * dy).sum() for s in (h, -h)]
            slope, formula = (at[0] - at[1]) / (2 * h), (got[name][0] * way).sum()
            assert abs(slope - formula) <= 1e-6 * (1 + abs(formula)), (name, float(slope), float(formula))

    x, w, b, r = d(3, 12, 5, 3), d(12), d(12), d(3, 12, 5, 3)
    for act in ("none", "leaky_relu", "silu"):
        agree(ref.group_norm_act, dict(x=x, weight=w, bias=b, residual=r),
              dict(dx="x", dweight="weight", dbias="bias", dresidual="residual"), d(3, 12, 5, 3), groups=4, eps=1e-3, act=act,
              slope=0.1)
    l, legal = d(4, 23), torch.rand(4, 23, generator=g) < 0.7
    hist = torch.randint(-1, 24, (4, 9), generator=g)
    for out in ("logits", "log_probs", "probs"):
        dy = torch.where(legal, d(4, 23), 0.0)

        def f(logits, bias, dy=None, **kw):
            got = ref.policy_logits(logits, legal, bias, hist, torch.tensor([9, 0, 4, 12]), 1.3, 0.25, 0.5, 0.75, out, torch.float64, dy)
            got["y"] = (torch.where(legal, got["y"][0], 0.0), None)
            return got
        agree(f, dict(logits=l, bias=d(23)), dict(dlogits="logits", dbias="bias"), dy)
        agree(f, dict(logits=l, bias=d(4, 23)), dict(dlogits="logits", dbias="bias"), dy)


def test_tensors_off_the_gpu_are_refused():
    from elf_amd import goenv, policy_ops
    x = torch.zeros(2, 8, 3, 3).to(memory_format=torch.channels_last)
    for call in (lambda: policy_ops.group_norm_act(x, 2), lambda: policy_ops.dropout(x, 0.5, torch.zeros(2, dtype=torch.int64)),
                 lambda: policy_ops.policy_logits(torch.zeros(2, 361)), lambda: policy_ops.policy_logits([1.0, 2.0])):
        with pytest.raises(goenv.GoEnvError, match="must be a tensor on the GPU"):
            call()


def _norm(**change):
    from elf_amd import goenv
    p = goenv.Norm(device=0, dtype=1, param_dtype=0, act=0, n=2, positions=9, channels=8, groups=2, eps=1e-5, slope=0.1,
                   x=256, x_sample=72, x_position=8, stats=256)
    for k, v in change.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("change,match", [
    (dict(dtype=3), "dtype must be"), (dict(dtype=-1), "dtype must be"), (dict(param_dtype=2), "param_dtype must be"),
    (dict(n=-1), "negative"), (dict(positions=-5), "negative"), (dict(channels=-8), "negative"), (dict(groups=3), "divide"),
    (dict(groups=0), "divide"), (dict(act=4), "act must be"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(eps=float("inf")), "eps"), (dict(act=2, slope=float("nan")), "slope"), (dict(x=None), "x is required"),
    (dict(x=257), "aligned"), (dict(weight=258), "aligned"), (dict(residual=255), "aligned")])
def test_norm_refusals(lib, change, match):
    p = _norm(**change)
    for rc in (lib.goenv_group_norm_act(C.byref(p), 256, None),
               lib.goenv_group_norm_act_grad(C.byref(p), 256, 72, 8, 256, None, None, None, None)):
        assert rc == -1 and match in lib.goenv_last_error().decode()


def test_norm_refusals_of_the_calls(lib):
    def says(rc, match):
        assert rc == -1 and match in lib.goenv_last_error().decode()
    says(lib.goenv_group_norm_act(None, 256, None), "p is NULL")
    says(lib.goenv_group_norm_act(C.byref(_norm()), None, None), "y is required")
    says(lib.goenv_group_norm_act(C.byref(_norm()), 257, None), "aligned")
    says(lib.goenv_group_norm_act_grad(C.byref(_norm(stats=None)), 256, 72, 8, 256, None, None, None, None), "stats")
    need = lib.goenv_group_norm_workspace(2, 9, 8, 2, 1, 1)
    assert need > 0
    for p in (_norm(), _norm(workspace=256, workspace_bytes=need - 1), _norm(workspace=264, workspace_bytes=need)):
        says(lib.goenv_group_norm_act_grad(C.byref(p), 256, 72, 8, 256, None, None, None, None), "workspace")
    p = _norm(workspace=256, workspace_bytes=need)
    says(lib.goenv_group_norm_act_grad(C.byref(p), None, 72, 8, 256, None, None, None, None), "dy is required")
    for empty in (dict(n=0), dict(positions=0), dict(channels=0)):
        assert lib.goenv_group_norm_act(C.byref(_norm(x=None, **empty)), None, None) == 0


@pytest.mark.parametrize("args,match", [
    ((0, 3, 8, 256, None, 256, 0.5, 256, 0, None), "dtype"), ((0, 0, -1, 256, None, 256, 0.5, 256, 0, None), "negative"),
    ((0, 0, 8, 256, None, 256, -0.1, 256, 0, None), "between 0 and 1"), ((0, 0, 8, 256, None, 256, 1.01, 256, 0, None), "between"),
    ((0, 0, 8, 256, None, 256, float("nan"), 256, 0, None), "between"), ((0, 0, 8, None, None, 256, 0.5, 256, 0, None), "required"),
    ((0, 0, 8, 256, None, None, 0.5, 256, 0, None), "required"), ((0, 0, 8, 256, None, 256, 0.5, None, 0, None), "required"),
    ((0, 0, 8, 258, None, 256, 0.5, 256, 0, None), "aligned"), ((0, 1, 8, 256, 257, 256, 0.5, 256, 0, None), "aligned"),
    ((0, 0, 8, 256, None, 256, 0.5, 260, 0, None), "aligned")])
def test_dropout_refusals(lib, args, match):
    assert lib.goenv_dropout(*args) == -1 and match in lib.goenv_last_error().decode()
    assert lib.goenv_dropout(0, 0, 0, None, None, None, 0.5, None, 0, None) == 0


def _rules(**change):
    from elf_amd import goenv
    p = goenv.LogitRules(device=0, dtype=1, out_dtype=0, out_kind=2, rows=2, cols=361, logits=256, logits_row=361, repetition=1.0,
                         temperature=1.0, stats=256)
    for k, v in change.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("change,match", [
    (dict(dtype=3), "dtype must be"), (dict(out_dtype=2), "out_dtype"), (dict(out_kind=3), "out_kind"), (dict(rows=-1), "range"),
    (dict(cols=-1), "range"), (dict(cols=1 << 31), "range"), (dict(legal=256, legal_bits=256), "not both"),
    (dict(bias=256, bias_dtype=2), "bias_dtype"), (dict(temperature=0.0), "temperature"), (dict(temperature=-1.0), "temperature"),
    (dict(temperature=float("inf")), "temperature"), (dict(temperature=float("nan")), "temperature"),
    (dict(temperature=2.0 ** -129), "temperature"), (dict(history=256, history_max=1, repetition=2.0 ** -129), "repetition"),
    (dict(history=256, history_max=-1), "history_max"), (dict(history=256, history_max=1, repetition=0.0), "repetition"),
    (dict(history=256, history_max=1, repetition=float("inf")), "repetition"),
    (dict(history=256, history_max=1, presence=float("nan")), "presence"),
    (dict(history=256, history_max=1, frequency=float("inf")), "frequency"), (dict(logits=None), "logits is required"),
    (dict(logits=257), "aligned"), (dict(legal_bits=257), "aligned"), (dict(history=260, history_max=1, history_i64=1), "aligned"),
    (dict(bias=258), "aligned")])
def test_logit_refusals(lib, change, match):
    p = _rules(**change)
    for rc in (lib.goenv_policy_logits(C.byref(p), 256, None), lib.goenv_policy_logits_grad(C.byref(p), 256, 361, 256, None, None)):
        assert rc == -1 and match in lib.goenv_last_error().decode()


def test_logit_refusals_of_the_calls(lib):
    def says(rc, match):
        assert rc == -1 and match in lib.goenv_last_error().decode()
    says(lib.goenv_policy_logits(None, 256, None), "p is NULL")
    says(lib.goenv_policy_logits(C.byref(_rules()), None, None), "out is required")
    says(lib.goenv_policy_logits(C.byref(_rules()), 258, None), "aligned")
    says(lib.goenv_policy_logits_grad(C.byref(_rules(stats=None)), 256, 361, 256, None, None), "stats")
    says(lib.goenv_policy_logits_grad(C.byref(_rules()), None, 361, 256, None, None), "d_out is required")
    says(lib.goenv_policy_logits_grad(C.byref(_rules()), 256, 361, 256, 256, None), "without a bias")
    need = lib.goenv_policy_logits_workspace(2, 361, 2, 1, 1)
    assert need > 0
    for p in (_rules(bias=256), _rules(bias=256, workspace=256, workspace_bytes=need - 1), _rules(bias=256, workspace=260, workspace_bytes=need)):
        says(lib.goenv_policy_logits_grad(C.byref(p), 256, 361, 256, 256, None), "workspace")
    for empty in (dict(rows=0), dict(cols=0)):
        assert lib.goenv_policy_logits(C.byref(_rules(logits=None, **empty)), None, None) == 0
