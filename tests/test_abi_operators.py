"""CPU-only checks of the sampling, scoring and optimiser entry points: what they refuse is refused on the host, before anything is
launched, also by a build of the host code under AddressSanitizer and UBSan."""
import ctypes
import math
import os
import subprocess
import sys

import pytest
import torch

from conftest import ROOT

FAKE = 0x1000  # never dereferenced: every call below fails validation first


class Tensor(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("param", "grad", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale", "step")] + [
        ("numel", ctypes.c_int64), ("dtype", ctypes.c_int32), ("state_bits", ctypes.c_int32), ("group", ctypes.c_int32), ("reserved", ctypes.c_int32)]


class Group(ctypes.Structure):
    _fields_ = [(n, ctypes.c_double) for n in ("lr", "beta1", "beta2", "eps", "weight_decay")] + [("d_lr", ctypes.c_void_p)]


def test_sample_tokens_refuses():
    from trl_amd import _lib

    def call(logits=FAKE, dtype=_lib.BF16, n_seq=2, rows=3, vocab=100, row_stride=100, uniform=FAKE, t=1.0, dt=None, k=0, p=1.0, dp=None,
             q=0.0, dq=None, ids=FAKE, ws=FAKE, ws_bytes=1 << 20):
        return _lib.lib.trlk_sample_tokens(logits, dtype, n_seq, rows, vocab, rows * row_stride, row_stride, uniform, 0, t, dt, k, None, p, dp,
                                           q, dq, None, 0, ids, FAKE, None, ws, ws_bytes, None)

    most = _lib.lib.trlk_token_filter_max_vocab()
    assert most >= 1 << 20
    assert call(dtype=7) == -3 and call(vocab=0) == -2 and call(n_seq=-1) == -2
    assert call(vocab=most + 1, row_stride=most + 1) == -7 and "vocab" in _lib.last_error()
    assert call(row_stride=99) == -4 and call(logits=None) == -1 and call(logits=FAKE + 1) == -4
    assert call(uniform=None) == -1 and call(ids=None) == -1
    for bad in (-1.0, math.nan, math.inf, 1e-320):
        assert call(t=bad) == -5 and "temperature" in _lib.last_error()
    for bad in (0.0, -0.5, 1.5, math.nan):
        assert call(p=bad) == -5 and "top_p" in _lib.last_error()
    for bad in (-0.5, 1.5, math.nan):
        assert call(q=bad) == -5 and "min_p" in _lib.last_error()
    need = _lib.lib.trlk_token_filter_workspace_bytes(6, 100, _lib.BF16)
    assert need > 0 and call(ws_bytes=need - 1) == -6 and call(ws=None) == -6 and call(ws=FAKE + 8) == -6
    assert call(n_seq=1 << 20, rows=1 << 20) == -2  # more rows than a launch has workgroups
    assert call(logits=None, n_seq=0) == 0 and _lib.last_error() == ""
    assert _lib.lib.trlk_token_filter_workspace_bytes(0, 100, 1) == 0
    assert _lib.lib.trlk_token_filter_workspace_bytes(5, most + 1, 1) == 0 and _lib.lib.trlk_token_filter_blocks(most + 1) == 0
    assert _lib.lib.trlk_token_filter_blocks(1) == 32 and _lib.lib.trlk_token_filter_blocks(2049) == 64


def test_filtered_logps_refuses():
    from trl_amd import _lib

    def fwd(logits=FAKE, dtype=_lib.F32, vocab=100, index=FAKE, t=1.0, p=1.0, state=FAKE, block_max=None, ws_bytes=1 << 20):
        return _lib.lib.trlk_filtered_logps_fwd(logits, dtype, 1, 3, vocab, 3 * vocab, vocab, index, t, None, 0, None, p, None, 0.0, None, None,
                                                FAKE, state, block_max, None, FAKE, ws_bytes, None)

    assert fwd(dtype=9) == -3 and fwd(vocab=-5) == -2 and fwd(index=None) == -1 and fwd(state=None) == -1 and fwd(t=-1.0) == -5
    assert fwd(p=2.0) == -5 and fwd(block_max=FAKE + 2) == -4 and fwd(ws_bytes=8) == -6 and fwd(logits=None) == -1

    def bwd(logits=FAKE, dtype=_lib.F32, t=1.0, state=FAKE, g=FAKE, out=FAKE, block_max=None):
        return _lib.lib.trlk_filtered_logps_bwd(logits, dtype, 1, 3, 100, 300, 100, FAKE, t, None, state, block_max, g, out, None)

    assert bwd(dtype=9) == -3 and bwd(logits=None) == -1 and bwd(t=math.nan) == -5 and bwd(state=None) == -1 and bwd(g=None) == -1
    assert bwd(out=None) == -1 and bwd(out=FAKE + 2) == -4 and bwd(block_max=FAKE + 1) == -4
    has = _lib.lib.trlk_token_filter_has_blocks
    assert has(1.0, None, 0, None, 1.0, None, 0.0, None) == 0
    assert [has(0.0, None, 0, None, 1.0, None, 0.0, None), has(1.0, FAKE, 0, None, 1.0, None, 0.0, None), has(1.0, None, 5, None, 1.0, None, 0.0, None),
            has(1.0, None, 0, FAKE, 1.0, None, 0.0, None), has(1.0, None, 0, None, 0.9, None, 0.0, None), has(1.0, None, 0, None, 1.0, FAKE, 0.0, None),
            has(1.0, None, 0, None, 1.0, None, 0.1, None), has(1.0, None, 0, None, 1.0, None, 0.0, FAKE)] == [1] * 8


def test_adamw_refuses():
    from trl_amd import _lib

    assert ctypes.sizeof(Tensor) == 80 and ctypes.sizeof(Group) == 48

    def call(n=1, n_groups=1, max_norm=1.0, ws=FAKE, ws_bytes=1 << 20, tensors=True, group=None, **kw):
        t = Tensor(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 1000, _lib.BF16, 32, 0, 0)
        for k, v in kw.items():
            setattr(t, k, v)
        g = Group(1e-3, 0.9, 0.999, 1e-8, 0.0, None)
        for k, v in (group or {}).items():
            setattr(g, k, v)
        return _lib.lib.trlk_adamw_step(ctypes.addressof(t) if tensors else None, n, ctypes.addressof(g), n_groups, max_norm, 0, FAKE, ws, ws_bytes, None)

    assert call(tensors=False) == -1 and call(n=-1) == -1
    for kw in (dict(dtype=5),):
        assert call(**kw) == -3
    for kw in (dict(state_bits=16), dict(group={"beta1": 1.0}), dict(group={"beta2": -0.1}), dict(group={"eps": -1.0}), dict(group={"lr": -1.0}),
               dict(group={"lr": math.nan}), dict(group={"weight_decay": -1.0}), dict(max_norm=math.nan), dict(n_groups=0)):
        assert call(**kw) == -5, kw
    for kw in (dict(param=None), dict(grad=None), dict(exp_avg=None), dict(exp_avg_sq=None), dict(step=None), dict(state_bits=8, exp_avg_scale=None)):
        assert call(**kw) == -1, kw
    assert call(numel=-1) == -2 and call(param=FAKE + 1) == -4 and call(exp_avg=FAKE + 2) == -4
    assert call(ws_bytes=16) == -6 and call(ws=FAKE + 8) == -6 and call(ws=None) == -6
    assert _lib.lib.trlk_adamw_step(None, 0, None, 0, -1.0, 0, None, None, 0, None) == 0
    values = _lib.lib.trlk_adamw_state_values
    assert values(FAKE, FAKE, -1, 1, FAKE, None) == -2 and values(None, FAKE, 5, 1, FAKE, None) == -1 and values(FAKE, FAKE, 5, 1, FAKE + 1, None) == -4
    assert values(None, None, 0, 1, None, None) == 0


def test_cpu_tensors_are_refused():
    import trl_amd

    x, u, ids = torch.randn(2, 16), torch.rand(2), torch.zeros(2, dtype=torch.long)
    with pytest.raises((NotImplementedError, RuntimeError)):
        trl_amd.sample_tokens(x, u)
    with pytest.raises((NotImplementedError, RuntimeError)):
        trl_amd.filtered_logps(x, ids)
    z = [torch.zeros(4)]
    with pytest.raises((NotImplementedError, RuntimeError)):
        trl_amd.adamw_step_(z, [torch.zeros(4)], [torch.zeros(4)], [torch.zeros(4)], [torch.zeros(())])
    w = torch.zeros(4, requires_grad=True)
    w.grad = torch.ones(4)
    with pytest.raises(RuntimeError, match="GPU"):
        trl_amd.AdamW([w]).step()
    # shapes are looked at before anything else
    for bad in (dict(uniforms=u[:1]), dict(uniforms=u, top_k=torch.zeros(3)), dict(uniforms=u, row_mask=torch.ones(3))):
        with pytest.raises(ValueError):
            trl_amd.sample_tokens(x, **bad)


def test_host_code_is_clean_under_asan_and_ubsan():
    from test_abi_sanitized import ASAN_LIB, _runtime

    if os.environ.get("TRLK_LIBRARY_PATH") == ASAN_LIB:
        pytest.skip("this is that run")
    if not os.path.exists(ASAN_LIB):
        pytest.skip("trl_amd/lib/libtrlk_asan.so is not built (make -C trl_amd/csrc asan)")
    runtime = _runtime()
    if runtime is None:
        pytest.skip("the sanitizer runtime of the ROCm clang is not installed")
    env = dict(os.environ)
    env["LD_PRELOAD"] = " ".join(p for p in (runtime, env.get("LD_PRELOAD", "")) if p)
    env["TRLK_LIBRARY_PATH"] = ASAN_LIB
    env["ASAN_OPTIONS"] = "detect_leaks=0:abort_on_error=0:exitcode=99"
    env["UBSAN_OPTIONS"] = "halt_on_error=1:print_stacktrace=1:exitcode=98"
    run = subprocess.run([sys.executable, "-m", "pytest", "-q", "-x", "-p", "no:cacheprovider", os.path.abspath(__file__)], env=env, cwd=ROOT,
                         capture_output=True, text=True, timeout=600)
    report = run.stdout[-3000:] + run.stderr[-3000:]
    assert run.returncode == 0, report
    assert "AddressSanitizer" not in report and "runtime error:" not in report, report
    assert " passed" in run.stdout


def test_launches_that_would_have_too_many_threads_are_refused():
    from trl_amd import _lib

    def sample(n_seq, rows, vocab):
        return _lib.lib.trlk_sample_tokens(FAKE, _lib.BF16, n_seq, rows, vocab, rows * vocab, vocab, FAKE, 0, 1.0, None, 0, None, 1.0, None, 0.0, None,
                                           None, 0, FAKE, FAKE, None, FAKE, 1 << 10, None)

    def grad(n_seq, rows, vocab):
        return _lib.lib.trlk_filtered_logps_bwd(FAKE, _lib.F32, n_seq, rows, vocab, rows * vocab, vocab, FAKE, 1.0, None, FAKE, None, FAKE, FAKE, None)

    for call in (sample, grad):
        for shape in ((1, 1 << 23, 8), (1 << 12, 1 << 11, 8), (1 << 62, 4, 8), (1, (1 << 26) // 76 + 1, 151936)):
            assert call(*shape) == -2 and "rows" in _lib.last_error()
    assert sample(1, (1 << 23) - 1, 8) == -6  # (rows that fit: the workspace does not)
    assert sample(1, (1 << 26) // 76 - 8, 151936) == -6
    t = Tensor(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, (1 << 34) + 1, _lib.BF16, 32, 0, 0)
    g = Group(1e-3, 0.9, 0.999, 1e-8, 0.0, None)
    step = lambda: _lib.lib.trlk_adamw_step(ctypes.addressof(t), 1, ctypes.addressof(g), 1, 1.0, 0, FAKE, FAKE, 16, None)  # noqa: E731
    assert step() == -2
    t.numel = 1 << 34
    assert step() == -6
    assert _lib.lib.trlk_adamw_state_values(FAKE, FAKE, (1 << 34) + 1, 1, FAKE, None) == -2


def test_block_maxima_are_read_by_vectors():
    """The caller's buffer of block maxima has the alignment that 16-byte loads of it need."""
    from trl_amd import _lib

    def fwd(dtype, block_max):
        return _lib.lib.trlk_filtered_logps_fwd(FAKE, dtype, 1, 3, 100, 300, 100, FAKE, 1.0, None, 5, None, 1.0, None, 0.0, None, None, FAKE, FAKE,
                                                block_max, None, FAKE, 8, None)

    for dtype in (_lib.F32, _lib.BF16, _lib.F16):
        for off in (2, 4, 8, 12):
            assert fwd(dtype, FAKE + off) == -4 and "block maxima" in _lib.last_error()
        assert fwd(dtype, FAKE) == -6 and fwd(dtype, FAKE + 16) == -6  # (aligned: the workspace is too small)


def test_temperatures_beyond_what_distances_in_fp32_bear():
    """Over 2^100 logits that are further apart than the largest fp32 number would both count."""
    from trl_amd import _lib

    def call(t, entry):
        if entry == "sample":
            return _lib.lib.trlk_sample_tokens(FAKE, _lib.F32, 1, 3, 100, 300, 100, FAKE, 0, t, None, 0, None, 0.9, None, 0.0, None, None, 0, FAKE, FAKE,
                                               None, FAKE, 8, None)
        if entry == "score":
            return _lib.lib.trlk_filtered_logps_fwd(FAKE, _lib.F32, 1, 3, 100, 300, 100, FAKE, t, None, 0, None, 0.9, None, 0.0, None, None, FAKE, FAKE,
                                                    None, None, FAKE, 8, None)
        return _lib.lib.trlk_filtered_logps_bwd(FAKE, _lib.F32, 1, 3, 100, 300, 100, FAKE, t, None, None, None, FAKE, FAKE, None)

    for entry, fine in (("sample", -6), ("score", -6), ("gradient", -1)):  # (the workspace is too small, an operand is missing)
        for t in (2.0**100 * (1 + 2.0**-52), 1.7e38, 1e300):
            assert call(t, entry) == -5 and "2^100" in _lib.last_error()
        assert call(2.0**100, entry) == fine and call(0.0, entry) == fine
