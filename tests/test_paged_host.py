"""Host side of the paged cache's and rotary calls, without a GPU."""

import math
import os
import random
import subprocess
import sys

import pytest
import torch

import foveated_kv_b200 as fkv
from foveated_kv_b200 import FkvNativeError, _native


def _step():
    """A small append on host tensors (its gradients are looked at first)."""
    rows = lambda h: torch.zeros(2, h, 64, dtype=torch.float16)
    pages = torch.zeros(3, 2, 16, 64, dtype=torch.float16)
    return dict(k=rows(2), v=rows(2), k_pages=pages, v_pages=pages.clone(), table=torch.zeros(2, 2, dtype=torch.int32),
                lens=torch.ones(2, dtype=torch.int32), q=rows(4), inv_freq=torch.zeros(32, dtype=torch.float64))


@pytest.mark.parametrize("name", ["k", "v", "q", "inv_freq"])
def test_gradients_are_refused(name):
    kw = _step()
    kw[name].requires_grad_()
    with pytest.raises(ValueError, match="gradient"):
        fkv.paged_append(**kw)
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
        fkv.paged_append(**kw)
    kw, ad = _step(), torch.autograd.forward_ad
    with ad.dual_level():
        kw[name] = ad.make_dual(kw[name], torch.ones_like(kw[name]))
        for mode in (torch.enable_grad, torch.no_grad):
            with mode(), pytest.raises(ValueError, match="forward gradient"):
                fkv.paged_append(**kw)
    with pytest.raises(ValueError, match="CUDA"):                # the tangent is gone with its level
        fkv.paged_append(**kw)


def _places(t):
    """Byte addresses of a tensor's elements, relative to its storage, with repeats."""
    at = torch.tensor([t.storage_offset()])
    for n, s in zip(t.shape, t.stride()):
        at = (at[:, None] + torch.arange(n) * s).reshape(-1)
    return (at[:, None] * t.element_size() + torch.arange(t.element_size())).reshape(-1).tolist()


def test_shared_memory_of_random_views():
    """The overlap test of the calls against the addresses themselves."""
    rng, share = random.Random(1), _native.ops().share_memory
    store = torch.zeros(400, dtype=torch.int32)
    kinds = [0, 0]
    for i in range(3000):
        views = []
        for j in range(2):
            base = store if rng.random() < 0.7 else store.view(torch.int16)
            dims = rng.randint(0, 4)
            steps = [rng.choice([1, 2, 3, 4, 6, 8, 12, 16, 24, 40]) for _ in range(dims)]
            if j and rng.random() < 0.5:
                base, steps = first
                dims = len(steps)
            first = base, steps
            shape = [rng.randint(1, 4) for _ in range(dims)]
            if rng.random() < 0.03 and dims:
                steps[0] = 0
            if rng.random() < 0.02 and dims:
                shape[-1] = 0
            views.append(base.as_strided(shape, steps, rng.randint(0, 60)))
        a, b = map(_places, views)
        assert share(*views) == share(*views[::-1]) == bool(set(a) & set(b)), [(v.shape, v.stride(), v.storage_offset()) for v in views]
        assert share(views[0], None) == (len(set(a)) < len(a)), [(v.shape, v.stride()) for v in views]
        kinds[bool(set(a) & set(b))] += 1
    assert min(kinds) > 500


def test_shared_memory_of_packed_rows():
    """Heads side by side in packed rows, however many: apart, and a view that is shifted: not."""
    share = _native.ops().share_memory
    qkv = torch.empty(100000, 48, 128, dtype=torch.float16)
    q, k, v = qkv[:, :32], qkv[:, 32:40], qkv[:, 40:]
    for a, b in ((q, k), (k, v), (v, q)):
        assert not share(a, b) and not share(b, a)
    assert share(qkv[:, 1:33], q) and share(qkv[:, 31:33], k) and not share(qkv[:, :32, :64], qkv[:, :32, 64:])
    assert share(q[1:], q[:-1]) and not share(q[50000:], q[:50000])
    t = qkv.view(10, 10000, 48, 128).transpose(1, 2)             # (B, H, S, D)
    assert not share(t[:, :32], t[:, 32:]) and share(t[:, :33], t[:, 32:]) and not share(t, None)
    assert not share(q, None) and not share(qkv[:, ::2], None)
    assert share(qkv.view(-1).as_strided((100, 4, 128), (512, 64, 1)), None)   # heads of 128 every 64
    assert share(qkv[:, :1].expand(-1, 4, -1), None)
    assert not share(torch.empty(0), torch.empty(0)) and not share(torch.empty(0), None)


CSRC = os.path.join(os.path.dirname(fkv.__file__), "csrc")


def _make(*args):
    r = subprocess.run(["make", "-C", CSRC, *args], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr
    return r.stdout


def test_the_c_library_builds_without_torch():
    """The default target wants nvcc alone, whatever the interpreter is."""
    out = _make("-n", "-B", "PY=/bin/false")
    assert "libfkv.so" in out and "ops.cpp" not in out and "torch" not in out
    out = _make("-n", "-B", f"PY={sys.executable}", "python")
    assert "libfkv.so" in out and "ops.cpp" in out and "-ltorch" in out


def test_the_python_calls_are_rebuilt_for_another_torch(tmp_path):
    """fkv_ops.so is out of date when the interpreter or its torch is another one."""
    ops, abi, ran = tmp_path / "fkv_ops.so", tmp_path / "python_abi", tmp_path / "ran"
    compiler = f"touch {ran}; touch {ops}; true"                 # in the compiler's place

    def rebuilt():
        ran.unlink(missing_ok=True)
        _make(str(ops), f"OPS={ops}", f"BUILD={tmp_path}", f"PY={sys.executable}", f"GXX={compiler}")
        return ran.exists()

    assert rebuilt() and torch.__version__ in abi.read_text()
    assert not rebuilt() and not rebuilt()
    abi.write_text(abi.read_text().replace(torch.__version__, "1.0.0"))
    assert rebuilt() and torch.__version__ in abi.read_text() and not rebuilt()


def test_the_python_calls_refuse_another_torch(monkeypatch):
    assert _native.ops().built_for.startswith("torch " + torch.__version__.split("+")[0])
    monkeypatch.setattr(_native, "_ops", None)
    monkeypatch.setattr(torch, "__version__", "99.1.0+other")
    with pytest.raises(FkvNativeError, match="this is torch 99.1.0.*rebuild"):
        _native.ops()
    monkeypatch.undo()
    assert _native.ops()


@pytest.mark.parametrize("rot,base,length,factor,slow,fast", [(128, 10000.0, 4096, 8.0, 1.0, 32.0), (64, 1e6, 32768, 4.0, 2.0, 20.0)])
def test_yarn_ramp_is_linear_in_the_turns(rot, base, length, factor, slow, fast):
    """Pair by pair against the formula, the pairs between the two ends among them."""
    f, amplitude = fkv.rotary_frequencies(rot, base, scaling="yarn", factor=factor, original_len=length,
                                          slow_turns=slow, fast_turns=fast, device="cpu")
    between = 0
    for p in range(rot // 2):
        plain = base ** (-2.0 * p / rot)
        turns = length * plain / (2 * math.pi)
        keep = min(1.0, max(0.0, (turns - slow) / (fast - slow)))
        between += 0.0 < keep < 1.0
        assert f[p].item() == pytest.approx(plain * keep + plain / factor * (1 - keep), rel=1e-12)
    assert between > 5 and amplitude == pytest.approx(0.1 * math.log(factor) + 1)


def test_a_step_that_fails_takes_nothing(monkeypatch):
    """extend whose copy to the device fails leaves pages, lengths and the step as they were."""
    c = fkv.PagedKVCache(1, 6, 2, 64, page=8, max_seqs=2, max_len=40, device="cpu")
    send = lambda values, dtype: torch.tensor(values, dtype=dtype)      # without pinned memory
    monkeypatch.setattr(c, "_send", send)
    c.extend([9, 3])
    for fails in (1, 2):                                                # the page numbers, the lengths
        def broken(values, dtype, left=[fails]):
            left[0] -= 1
            if left[0] == 0:
                raise RuntimeError("out of memory")
            return send(values, dtype)
        monkeypatch.setattr(c, "_send", broken)
        with pytest.raises(RuntimeError, match="out of memory"):
            c.extend([20, 1])
        assert c.free_pages == 3 and c.lengths == [9, 3] and c.lens.tolist() == [9, 3]
    monkeypatch.setattr(c, "_send", send)
    c.extend([20, 1])
    rows = c.table.tolist()
    assert c.lengths == [29, 4] and c.free_pages == 1
    assert sorted(rows[0][:4] + rows[1][:1] + c._free) == list(range(6)) and rows[0][4] == rows[1][1] == -1
    c.release(0)
    assert c.free_pages == 5
