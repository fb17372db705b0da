"""CPU: the policy operators' C-ABI (include/contracts_policy.h) exports what it declares, its structs are the ctypes mirrors', it refuses
every bad argument before anything is launched, and it never falls back to a CPU path."""
import ctypes as C
import os
import re
import subprocess
import tempfile

import numpy as np
import pytest
import torch

import policy_oracle as oracle

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "contracts_policy.h")
EINVAL, ENODEV = -22, -19
FAKE = 1 << 20  # an aligned address that no check reads


@pytest.fixture(scope="module")
def L():
    from contracts_amd import _lib
    return _lib.load_policy()


def test_header_functions_exported(L):
    from contracts_amd import _lib
    src = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    names = set(re.findall(r"\b(ce_[a-z0-9_]+)\s*\(", src))
    assert names == set(_lib.POLICY_EXPORTS)
    assert L.ce_policy_abi_version() == _lib.POLICY_ABI_VERSION


def test_struct_layout_matches_ctypes():
    from contracts_amd import _lib
    structs = {"ce_scan": _lib.CeScan, "ce_scan_grad": _lib.CeScanGrad, "ce_advantage": _lib.CeAdvantage, "ce_logits": _lib.CeLogits, "ce_logits_grad": _lib.CeLogitsGrad}
    lines, want = [], []
    for name, cls in structs.items():
        lines.append('printf("%%zu ", sizeof(%s));' % name)
        want.append(C.sizeof(cls))
        for f, _ in cls._fields_:
            lines.append('printf("%%zu ", offsetof(%s, %s));' % (name, f))
            want.append(getattr(cls, f).offset)
    with tempfile.TemporaryDirectory() as d:
        src, exe = os.path.join(d, "t.c"), os.path.join(d, "t")
        open(src, "w").write('#include <stdio.h>\n#include <stddef.h>\n#include "contracts_policy.h"\nint main(void) { %s return 0; }' % " ".join(lines))
        subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), src, "-o", exe])
        assert [int(v) for v in subprocess.check_output([exe]).split()] == want


def _scan(**kw):
    from contracts_amd import _lib
    f = dict(abi_version=1, dtype=_lib.F32, gate_dtype=_lib.F32, steps=4, rows=3, channels=6, heads=2, x_step=18, x_row=6, gate_step=6, gate_row=2, x=FAKE, gate=FAKE,
             y=FAKE, last=FAKE)
    f.update(kw)
    return _lib.CeScan(**f)


@pytest.mark.parametrize("kw,word", [
    (dict(abi_version=7), "abi_version"), (dict(dtype=4), "x must be"), (dict(dtype=1, gate_dtype=2), "gate must be"), (dict(gate_dtype=1), "gate must be"),
    (dict(dtype=3, gate_dtype=0), "gate must be"), (dict(flags=2), "flags"), (dict(heads=4), "divide"), (dict(heads=0), "divide"), (dict(heads=12), "divide"),
    (dict(rows=1 << 20, channels=1 << 10, heads=1), "columns"), (dict(rows=1 << 40), "columns"), (dict(steps=1 << 60), "elements"), (dict(x=None), "null"), (dict(y=None), "null"),
    (dict(x=FAKE + 2), "aligned"), (dict(gate=FAKE + 1), "aligned"), (dict(last=FAKE + 2), "aligned"), (dict(x_row=-6), "far apart"), (dict(gate_row=1 << 27), "far apart"),
    (dict(gate=None, decay=float("nan")), "finite"),
    (dict(gate=None, decay=float("inf")), "finite")])
def test_scan_refusals(L, kw, word):
    s, nbytes = _scan(**kw), C.c_uint64()
    assert L.ce_linear_scan(C.byref(s), None) == EINVAL and word in L.ce_policy_error().decode()
    assert L.ce_linear_scan_workspace(C.byref(s), C.byref(nbytes)) == EINVAL
    assert L.ce_linear_scan(None, None) == EINVAL and L.ce_linear_scan_workspace(C.byref(_scan()), None) == EINVAL


def test_scan_backward_refusals(L):
    from contracts_amd import _lib
    g, nbytes = _lib.CeScanGrad(dy=FAKE, dlast=FAKE, dx=FAKE, dgate=FAKE, dstate=FAKE), C.c_uint64()
    assert L.ce_linear_scan_backward(C.byref(_scan()), None, None) == EINVAL and L.ce_linear_scan_backward(None, C.byref(g), None) == EINVAL
    for s, word in ((_scan(), "saved"), (_scan(saved=FAKE, dtype=3, gate_dtype=3), "double"), (_scan(saved=FAKE, gate=None, decay=0.5), "constant gate")):
        assert L.ce_linear_scan_backward(C.byref(s), C.byref(g), None) == EINVAL and word in L.ce_policy_error().decode()
    g.dx = FAKE + 1
    assert L.ce_linear_scan_backward_workspace(C.byref(_scan(saved=FAKE)), C.byref(g), C.byref(nbytes)) == EINVAL and b"aligned" in L.ce_policy_error()


def test_scan_asks_for_a_workspace_only_where_time_is_split(L):
    nbytes = C.c_uint64()
    for kw, split in ((dict(), False), (dict(steps=5000), True), (dict(steps=5000, rows=20000), False)):
        assert L.ce_linear_scan_workspace(C.byref(_scan(**kw)), C.byref(nbytes)) == 0 and (nbytes.value > 0) == split
    s = _scan(steps=5000)
    assert L.ce_linear_scan_workspace(C.byref(s), C.byref(nbytes)) == 0
    s.workspace, s.workspace_bytes = FAKE, nbytes.value - 1
    assert L.ce_linear_scan(C.byref(s), None) == EINVAL and b"workspace" in L.ce_policy_error()
    s.state = s.last  # moved on in place: the time axis stays whole
    assert L.ce_linear_scan_workspace(C.byref(s), C.byref(nbytes)) == 0 and nbytes.value == 0


@pytest.mark.parametrize("kw,word", [
    (dict(abi_version=0), "abi_version"), (dict(reward_dtype=1), "reward"), (dict(value_dtype=3), "value"), (dict(flags=2), "flags"), (dict(first_plane=4), "first_plane"),
    (dict(gamma=float("nan")), "finite"), (dict(lam=float("inf")), "finite"), (dict(reward=None), "null"), (dict(advantage=None, ret=None), "null"), (dict(reward=FAKE + 4), "aligned"),
    (dict(rows=1 << 29), "columns"), (dict(planes=1 << 60), "elements")])
def test_advantages_refusals(L, kw, word):
    from contracts_amd import _lib
    f = dict(abi_version=1, reward_dtype=_lib.F64, value_dtype=_lib.F32, planes=4, rows=3, agents=2, gamma=0.9, lam=0.9, reward=FAKE, value=FAKE, advantage=FAKE, ret=FAKE)
    a = _lib.CeAdvantage(**dict(f, **kw))
    assert L.ce_advantages(C.byref(a), None) == EINVAL and word in L.ce_policy_error().decode()
    assert L.ce_advantages(None, None) == EINVAL


def _logits(**kw):
    from contracts_amd import _lib
    f = dict(abi_version=1, dtype=_lib.F32, out_dtype=_lib.F32, rows=6, vocab=10, logits_row=10, out_row=10, logits=FAKE, out=FAKE, repetition_all=1.0)
    return _lib.CeLogits(**dict(f, **kw))


@pytest.mark.parametrize("kw,word", [
    (dict(abi_version=2), "abi_version"), (dict(dtype=3), "logits"), (dict(out_dtype=1), "output"), (dict(rows=1 << 24), "rows"), (dict(vocab=1 << 29), "tokens"),
    (dict(history=1 << 31), "history"), (dict(logits=None), "null"), (dict(out=None), "null"), (dict(out=FAKE + 2), "aligned"), (dict(tokens=FAKE, token_dtype=0, history=3), "tokens"),
    (dict(tokens=FAKE + 1, token_dtype=5, history=3), "aligned"), (dict(tokens=FAKE, token_dtype=5, history=3, repetition_all=0.0), "positive"),
    (dict(tokens=FAKE, token_dtype=5, history=3, repetition_all=float("nan")), "positive"), (dict(tokens=FAKE, token_dtype=5, history=3, presence_all=float("inf")), "finite"),
    (dict(lengths=FAKE), "without tokens"), (dict(bias=FAKE, bias_dtype=1, bias_rows=1), "bias"), (dict(bias=FAKE, bias_dtype=0, bias_rows=4), "divide"),
    (dict(bias=FAKE, bias_dtype=0, bias_rows=0), "divide"), (dict(mask=FAKE, mask_dtype=0, mask_rows=1), "mask"), (dict(mask=FAKE, mask_dtype=4, mask_rows=5), "divide"),
    (dict(mask=FAKE, mask_dtype=5, mask_rows=0, mask_index=FAKE), "mask_rows"), (dict(mask_index=FAKE), "without a mask"), (dict(logits_row=12), "in place"),
    (dict(out_row=9), "overlap"), (dict(out_row=0), "overlap"), (dict(out_row=-9), "overlap")])
def test_logits_refusals(L, kw, word):
    s = _logits(**kw)
    assert L.ce_process_logits(C.byref(s), None) == EINVAL and word in L.ce_policy_error().decode()
    assert L.ce_process_logits(None, None) == EINVAL


def test_logits_backward_refusals(L):
    from contracts_amd import _lib
    nbytes = C.c_uint64()
    s = _logits(bias=FAKE, bias_dtype=0, bias_rows=2)
    assert L.ce_process_logits_backward(C.byref(s), None, None) == EINVAL
    for g, word in ((_lib.CeLogitsGrad(dlogits=FAKE), "null"), (_lib.CeLogitsGrad(dout=FAKE, dlogits=FAKE + 1), "aligned"), (_lib.CeLogitsGrad(dout=FAKE, dbias=FAKE), "workspace")):
        assert L.ce_process_logits_backward(C.byref(s), C.byref(g), None) == EINVAL and word in L.ce_policy_error().decode()
    g = _lib.CeLogitsGrad(dout=FAKE, dbias=FAKE)
    assert L.ce_process_logits_backward(C.byref(_logits()), C.byref(g), None) == EINVAL and b"without a bias" in L.ce_policy_error()
    assert L.ce_process_logits_backward_workspace(C.byref(s), C.byref(g), C.byref(nbytes)) == 0 and nbytes.value >= 2 * 10 * 4


def test_empty_calls_need_no_device(L):
    from contracts_amd import _lib
    assert L.ce_linear_scan(C.byref(_scan(rows=0)), None) == 0 and L.ce_linear_scan(C.byref(_scan(steps=0, x=None, y=None, last=None)), None) == 0
    assert L.ce_process_logits(C.byref(_logits(rows=0)), None) == 0 and L.ce_process_logits(C.byref(_logits(vocab=0)), None) == 0
    assert L.ce_advantages(C.byref(_lib.CeAdvantage(abi_version=1, reward_dtype=3, planes=0)), None) == 0


def test_no_gpu_fails_loudly(L):
    from contracts_amd import policy_ops as ops
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    assert L.ce_linear_scan(C.byref(_scan()), None) == ENODEV and L.ce_process_logits(C.byref(_logits()), None) == ENODEV
    x = torch.zeros(2, 3, 4)
    for call in (lambda: ops.linear_scan(x, 0.5), lambda: ops.advantages(x, x), lambda: ops.process_logits(x)):
        with pytest.raises(ValueError, match="no CPU path"):
            call()


def test_pack_mask_and_the_oracles_gradients():
    from contracts_amd import policy_ops as ops
    g = torch.Generator().manual_seed(3)
    for V in (1, 31, 32, 33, 151):
        m = torch.rand((3, V), generator=g) < 0.5
        w, v = ops.pack_mask(m), torch.arange(V)
        assert w.dtype == torch.int32 and w.shape == (3, (V + 31) // 32) and (((w[:, v // 32].long() >> (v % 32)) & 1) != 0).equal(m)
    # the formulas of the oracle's gradients, against differences of its values (multilinear in each gate: central differences are exact)
    x, a, s = torch.randn((5, 2, 4), generator=g).double(), torch.rand((5, 2, 2), generator=g).double(), torch.randn((2, 4), generator=g).double()
    done, dy, dl = torch.rand((5, 2), generator=g) < 0.3, torch.randn((5, 2, 4), generator=g).double(), torch.randn((2, 4), generator=g).double()
    for reverse in (False, True):
        def value():
            f = oracle.scan(x, a, s, done, reverse)
            return (f["y"] * dy.numpy()).sum() + (f["last"] * dl.numpy()).sum()
        got = oracle.scan_grad(oracle.scan(x, a, s, done, reverse), dy, dl, 2, reverse)
        for t, d in ((x, got["dx"]), (a, got["dgate"]), (s, got["dstate"])):
            flat = t.view(-1)
            for i in range(flat.numel()):
                keep = flat[i].item()
                flat[i] = keep + 0.25
                up = value()
                flat[i] = keep - 0.25
                down = value()
                flat[i] = keep
                assert abs((up - down) / 0.5 - d.reshape(-1)[i]) < 1e-12 * (1 + np.abs(d).max()) * 100


def test_tracers_transforms_and_wrapped_tensors_are_refused():
    """a call is no operation that they could record: the graph would hold the outputs' allocation alone"""
    from torch._subclasses import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx

    from contracts_amd import policy_ops as ops
    x = torch.zeros(2, 3, 4)

    class Wrapper(torch.Tensor):
        @staticmethod
        def __new__(cls, inner):
            return torch.Tensor._make_wrapper_subclass(cls, inner.size(), dtype=inner.dtype)

        @classmethod
        def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
            raise AssertionError("never reached")

    for call in (lambda t: ops.linear_scan(t, 0.5)[0], lambda t: ops.advantages(t, t)[0], lambda t: ops.process_logits(t)):
        with pytest.raises(ValueError, match="traced"):
            torch.jit.trace(call, x)
        for mode in ("real", "fake"):
            with pytest.raises(ValueError, match="traced"):
                make_fx(call, tracing_mode=mode)(x)
        with FakeTensorMode(), pytest.raises(ValueError, match="traced"):
            call(torch.empty(2, 3, 4))
        with FakeTensorMode():
            fake = torch.empty(2, 3, 4)
        for run in (lambda: torch.vmap(call)(x.expand(2, 2, 3, 4)), lambda: torch.func.grad(lambda t: call(t).sum())(x), lambda: call(fake), lambda: call(torch._efficientzerotensor(2, 3, 4)),
                    lambda: call(Wrapper(x))):
            with pytest.raises(ValueError, match="wrapped"):
                run()
        with pytest.raises(ValueError, match="no CPU path"):
            call(torch.nn.Parameter(x))


def test_scalars_are_checked_as_the_kernels_hold_them(L):
    """finite and positive as a double is not enough where float arithmetic follows: what becomes 0 or infinite there is refused"""
    from contracts_amd import _lib
    nbytes = C.c_uint64()
    for value in (1e-50, 2.0 ** -127, 1e-39, 2.0 ** 126 * 1.0001, 1e39, 1e300):
        s = _logits(tokens=FAKE, token_dtype=5, history=3, repetition_all=value)
        assert L.ce_process_logits(C.byref(s), None) == EINVAL and b"repetition must be positive" in L.ce_policy_error()
    for kw in (dict(presence_all=1e39), dict(frequency_all=-1e300)):
        s = _logits(tokens=FAKE, token_dtype=5, history=3, **kw)
        assert L.ce_process_logits(C.byref(s), None) == EINVAL and b"finite" in L.ce_policy_error()
    g = _lib.CeLogitsGrad(dout=FAKE, dlogits=FAKE + 4096)
    for kw in (dict(repetition_all=2.0 ** -126), dict(repetition_all=2.0 ** 126), dict(presence_all=-3e38), dict(repetition=FAKE, repetition_all=0.0)):  # (a call that launches nothing)
        assert L.ce_process_logits_backward_workspace(C.byref(_logits(tokens=FAKE, token_dtype=5, history=3, **kw)), C.byref(g), C.byref(nbytes)) == 0
    for dtype, ok in ((_lib.F32, 3e38), (_lib.BF16, 3e38), (_lib.F64, 1e300)):
        for decay, fine in ((ok, True), (1e39, dtype == _lib.F64), (-1e39, dtype == _lib.F64), (float("inf"), False)):
            rc = L.ce_linear_scan_workspace(C.byref(_scan(dtype=dtype, gate_dtype=dtype, gate=None, decay=decay)), C.byref(nbytes))
            assert rc == (0 if fine else EINVAL) and (fine or b"finite" in L.ce_policy_error())
    f = dict(abi_version=1, reward_dtype=_lib.F64, value_dtype=_lib.F32, planes=4, rows=3, agents=2, reward=FAKE, value=FAKE, advantage=FAKE, ret=FAKE)
    assert L.ce_advantages(C.byref(_lib.CeAdvantage(gamma=1e200, lam=1e200, **f)), None) == EINVAL and b"finite" in L.ce_policy_error()


def test_logits_gradients_do_not_overlap_what_they_are_made_of(L):
    """dlogits is written before the scores under a repetition penalty are read again: not over dout, nor over the logits"""
    from contracts_amd import _lib
    nbytes, size, far = C.c_uint64(), 6 * 10 * 4, FAKE + 8192
    for dout, logits, dlogits, fine in ((FAKE, far, FAKE, False), (FAKE, far, far, False), (FAKE, far, FAKE + size - 4, False), (FAKE, far, far - size + 4, False), (FAKE, far, FAKE + size, True),
                                        (FAKE, far, far - size, True), (FAKE, far, far + size, True)):
        s, g = _logits(tokens=FAKE, token_dtype=5, history=3, logits=logits), _lib.CeLogitsGrad(dout=dout, dout_row=10, dlogits=dlogits)
        assert L.ce_process_logits_backward_workspace(C.byref(s), C.byref(g), C.byref(nbytes)) == (0 if fine else EINVAL)
        if not fine:
            assert b"overlaps" in L.ce_policy_error() and L.ce_process_logits_backward(C.byref(s), C.byref(g), None) == EINVAL
    # rows apart, backwards or shared: what lies between the first and the last counts
    for row, reach in ((20, 5 * 20 + 10), (0, 10), (-20, 10)):
        s, g = _logits(logits=far), _lib.CeLogitsGrad(dout=FAKE + 4096, dout_row=row, dlogits=FAKE + 4096 + 4 * reach)
        assert L.ce_process_logits_backward_workspace(C.byref(s), C.byref(g), C.byref(nbytes)) == 0
        g.dlogits -= 4
        assert L.ce_process_logits_backward_workspace(C.byref(s), C.byref(g), C.byref(nbytes)) == EINVAL


def test_pack_mask_takes_what_the_masks_of_bytes_take():
    """nonzero = allowed, as process_logits reads a uint8 mask: a byte of 2 or 255 is one bit, its own"""
    from contracts_amd import policy_ops as ops
    m = torch.randint(0, 256, (3, 70), generator=torch.Generator().manual_seed(1)).to(torch.uint8)
    m[:, ::3] = 0
    assert ops.pack_mask(m).equal(ops.pack_mask(m != 0))
