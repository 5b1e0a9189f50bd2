"""CPU: what the policy-network operators refuse before they reach a device (elf_amd/policy_ops.py, include/goenv.h)."""
import ctypes as C

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from elf_amd import goenv
    return goenv.load_library()


def rules(**change):
    from elf_amd import goenv
    p = goenv.LogitRules(device=0, dtype=1, out_dtype=0, out_kind=2, rows=2, cols=361, logits=256, logits_row=361, repetition=1.0,
                         temperature=1.0, stats=256, legal_row=361, bits_row=12, history_row=4)
    for k, v in change.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("change,args,match", [
    (dict(rows=-1), (256, None, None), "range"), (dict(cols=(1 << 28) + 1), (256, None, None), "range"),
    (dict(legal=256, legal_bits=256), (256, None, None), "not both"), (dict(history=256, history_max=-1), (None, 256, None), "history_max"),
    (dict(), (256, None, None), "does not have"), (dict(legal=256), (None, 256, None), "does not have"),
    (dict(history=256, history_max=2), (None, 256, 256), "does not have"), (dict(legal=256), (258, None, None), "aligned"),
    (dict(history=256, history_max=2, history_i64=1), (None, 260, None), "aligned"),
    (dict(history=260, history_max=2, history_i64=1), (None, 256, None), "aligned"), (dict(legal_bits=257), (256, None, None), "aligned")])
def test_refused_copies_of_rules(lib, change, args, match):
    assert lib.goenv_policy_logits_keep(C.byref(rules(**change)), *args, None) == -1 and match in lib.goenv_last_error().decode()
    assert lib.goenv_policy_logits_keep(None, *args, None) == -1 and "NULL" in lib.goenv_last_error().decode()


def test_nothing_to_copy_is_no_error(lib):
    for change in (dict(rows=0, legal=256), dict(cols=0, legal=256), dict(legal=256, history=256, history_max=0)):
        args = (256 if "rows" in change or "cols" in change else None, 256 if "history" in change else None, None)
        assert lib.goenv_policy_logits_keep(C.byref(rules(**change)), *args, None) == 0


def operators():
    """{name: call of (tensor)} of arguments that pass every check but that of the device."""
    from elf_amd import policy_ops
    rng = torch.zeros(2, dtype=torch.int64)
    return {"group_norm_act": lambda x: policy_ops.group_norm_act(x.t(), 2), "dropout": lambda x: policy_ops.dropout(x, 0.5, rng),
            "policy_logits": lambda x: policy_ops.policy_logits(x)}


@pytest.mark.parametrize("name", ["group_norm_act", "dropout", "policy_logits"])
def test_forward_mode_derivatives_are_refused(name):
    import torch.autograd.forward_ad as forward_ad
    from elf_amd import goenv
    call, x = operators()[name], torch.ones(8, 6)
    with forward_ad.dual_level():
        with pytest.raises(goenv.GoEnvError, match="forward-mode"):
            call(forward_ad.make_dual(x, torch.ones_like(x)))
        with pytest.raises(goenv.GoEnvError, match="on the GPU"):
            call(x)


@pytest.mark.parametrize("name", ["group_norm_act", "dropout", "policy_logits"])
def test_calls_under_a_trace_are_refused(name):
    from torch.fx.experimental.proxy_tensor import make_fx
    from elf_amd import goenv
    call, x = operators()[name], torch.ones(8, 6)
    with pytest.raises(goenv.GoEnvError, match="trace"):
        torch.jit.trace(call, (x,), check_trace=False)
    for mode in ("real", "fake"):
        with pytest.raises(goenv.GoEnvError, match="trace"):
            make_fx(call, tracing_mode=mode)(x)
    with pytest.raises(goenv.GoEnvError, match="on the GPU"):
        call(x)


class Wrapper(torch.Tensor):
    """A tensor with a type and sizes that holds another one and no memory of its own."""
    @staticmethod
    def __new__(cls, t):
        return torch.Tensor._make_wrapper_subclass(cls, t.size(), strides=t.stride(), dtype=t.dtype, device=t.device)

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise AssertionError(func)


def test_tensors_without_memory_are_refused():
    from elf_amd import goenv, policy_ops
    x = torch.ones(6, 8)
    for other in (Wrapper(x), torch._efficientzerotensor(6, 8)):
        for call in (lambda t: policy_ops.group_norm_act(t, 2), lambda t: policy_ops.dropout(t, 0.5, torch.zeros(2, dtype=torch.int64)),
                     policy_ops.policy_logits):
            with pytest.raises(goenv.GoEnvError, match="memory"):
                call(other)
    with pytest.raises(goenv.GoEnvError, match="on the GPU"):
        policy_ops.group_norm_act(x[:0], 2)


def test_no_number_of_rows_is_too_large_for_a_launch(lib):
    """They reach the selection of the device (there is no such device: nothing is launched)."""
    for change in (dict(rows=9_000_000, cols=2), dict(rows=1 << 33), dict(rows=1 << 20, cols=131072), dict(rows=3, cols=1 << 28)):
        for bias in ({}, dict(bias=256, bias_row=0)):
            p = rules(device=1 << 20, workspace=256, workspace_bytes=1 << 62, **change, **bias)
            for rc in (lib.goenv_policy_logits(C.byref(p), 256, None), lib.goenv_policy_logits_grad(C.byref(p), 256, p.cols, 256, 256 if bias else None, None)):
                assert rc == -1 and "selecting the device" in lib.goenv_last_error().decode()


@pytest.mark.parametrize("groups", [0, -8, 24, 256, 2.0])
def test_a_net_of_groups_that_do_not_divide_its_channels_is_refused(groups):
    """It would be a net of BatchNorm, or of another number of groups.  The heads (two channels and one) take what divides them."""
    from elf_amd.df_model import PolicyValueNet
    with pytest.raises(ValueError, match="groups"):
        PolicyValueNet(dim=128, num_block=1, norm="group", groups=groups)
    net = PolicyValueNet(dim=96, num_block=1, norm="group", groups=8)
    assert [net.init_conv[1].num_groups, net.pi_final_conv[1].num_groups, net.value_final_conv[1].num_groups] == [8, 2, 1]
    assert PolicyValueNet(dim=128, num_block=1, groups=groups).bn                         # not asked for: not looked at


@pytest.mark.parametrize("name", ["row_repetition", "row_presence", "row_frequency", "row_temperature", "stats", "history_len"])
def test_rows_that_are_not_aligned_are_refused(lib, name):
    """A scalar load drops the low bits of an address: it would be another row's value."""
    p = rules(device=1 << 20, history=256, history_max=4, workspace=256, workspace_bytes=1 << 40, **{name: 258})
    for rc in (lib.goenv_policy_logits(C.byref(p), 256, None), lib.goenv_policy_logits_grad(C.byref(p), 256, 361, 256, None, None)):
        assert rc == -1 and "aligned" in lib.goenv_last_error().decode()


def test_statistics_that_are_not_aligned_are_refused(lib):
    from elf_amd import goenv
    p = goenv.Norm(device=1 << 20, dtype=1, param_dtype=0, act=0, n=2, positions=9, channels=8, groups=2, eps=1e-5, x=256, x_sample=72, x_position=8,
                   stats=258, workspace=256, workspace_bytes=1 << 40)
    for rc in (lib.goenv_group_norm_act(C.byref(p), 256, None), lib.goenv_group_norm_act_grad(C.byref(p), 256, 72, 8, 256, None, None, None, None)):
        assert rc == -1 and "aligned" in lib.goenv_last_error().decode()
