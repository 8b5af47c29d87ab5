"""The layer operators without a GPU: the C ABI of include/ppo_layers.h, its
argument checks (which return before any device work), the Python refusals,
and the oracle they are tested against."""

import ctypes
import os
import re
import shutil
import subprocess

import numpy as np
import pytest
import torch

import ppo_amd
from oracle import layers_oracle as ref
from ppo_amd import _lib, layers

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "ppo_layers.h")
P = ctypes.c_void_p(4096)  # non-null, aligned, never dereferenced


def declared_functions():
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    return sorted(set(re.findall(r"\b(ppo_layer_[a-z0-9_]+)\s*\(", text)))


def test_exports_match_the_header():
    lib = _lib.load_layers()
    names = declared_functions()
    assert names and set(names) == set(_lib.LAYER_SIGNATURES)
    for name in names:
        assert hasattr(lib, name)
    syms = os.popen(f"nm -D --defined-only {_lib.LAYERS_PATH}").read()
    assert set(re.findall(r"\bT (\S+)$", syms, flags=re.M)) == set(names)


def test_loads_to_lds_wait_for_their_descriptor(tmp_path):
    """Five wait states lie between a vector instruction that writes a scalar
    register and a buffer load that reads it.  The loads to LDS are inline
    assembly, which the compiler's own hazard handling does not look into, so each
    block has to wait by itself, whatever stands before it."""
    objdump = "/opt/rocm/llvm/bin/llvm-objdump"
    if not os.path.exists(objdump):
        pytest.skip("no llvm-objdump")
    lib = shutil.copy(_lib.LAYERS_PATH, tmp_path)
    subprocess.run([objdump, "--offloading", lib], cwd=tmp_path, check=True, capture_output=True)
    loads = 0
    for name in os.listdir(tmp_path):
        if not name.endswith("gfx950") or os.path.getsize(tmp_path / name) == 0:
            continue
        text = subprocess.run([objdump, "-d", "--no-show-raw-insn", "--no-leading-addr",
                               str(tmp_path / name)], check=True, capture_output=True, text=True)
        code = [line.split("//")[0].split() for line in text.stdout.splitlines()]
        for i, words in enumerate(code):
            if not words or not words[0].startswith("buffer_load") or words[-1] != "lds":
                continue
            loads += 1
            states, j = 0, i - 1
            while code[j] and (code[j][0] == "s_nop" or code[j][:2] == ["s_mov_b32", "m0,"]):
                states += int(code[j][1]) + 1 if code[j][0] == "s_nop" else 1
                j -= 1
            assert states >= 5, f"{name}: {' '.join(words)} after {states} wait states"
    assert loads > 0


def drop(p, seed=1):
    return ctypes.byref(_lib.Dropout(p, seed, None, None))


def test_dropout_arguments():
    f = _lib.load_layers().ppo_layer_dropout
    assert f(P, P, 3, 4, 4, drop(0.1), None) == 1          # type
    assert f(P, P, 0, -1, 4, drop(0.1), None) == 1
    assert f(P, P, 0, 4, 4, None, None) == 1
    for p in (-0.1, 1.1, float("nan")):
        assert f(P, P, 0, 4, 4, drop(p), None) == 1
    assert f(None, P, 0, 4, 4, drop(0.1), None) == 1
    assert f(None, None, 0, 0, 4, drop(0.1), None) == 0    # nothing to do
    assert f(None, None, 0, 4, 0, drop(0.1), None) == 0
    assert f(P, P, 0, 1, (1 << 33) + 1, drop(0.1), None) == 3


def test_quantize_arguments():
    f = _lib.load_layers().ppo_layer_quantize_rows
    assert f(P, 5, 4, 4, P, P, None) == 1
    assert f(P, 0, 4, 0, P, P, None) == 1
    assert f(P, 0, 4, 4, None, P, None) == 1
    assert f(None, 0, 0, 4, None, None, None) == 0
    assert f(P, 0, 1 << 31, 4, P, P, None) == 3


def test_int8_linear_arguments():
    lib = _lib.load_layers()
    f = lib.ppo_layer_int8_linear

    def call(x=P, xq=None, xs=None, wq=P, ws=P, dtype=0, M=200, N=64, K=64, out=P, work=P,
             nbytes=1 << 40):
        return f(x, xq, xs, wq, ws, None, dtype, M, N, K, out, work, nbytes, None)

    assert call(dtype=-1) == 1 and call(M=-1) == 1 and call(N=0) == 1 and call(K=0) == 1
    assert call(wq=None) == 1 and call(ws=None) == 1 and call(out=None) == 1
    assert call(x=None) == 1 and call(x=None, xq=P) == 1
    assert call(M=0, x=None, wq=None, out=None, work=None) == 0
    assert call(K=(1 << 17) + 1) == 3
    need = lib.ppo_layer_int8_linear_workspace_bytes(200, 64, 64, 1)
    assert need >= 200 * 64 + 200 * 4
    assert call(nbytes=need - 1) == 2 and call(work=None) == 2
    assert call(work=ctypes.c_void_p(4097)) == 2
    assert lib.ppo_layer_int8_linear_workspace_bytes(0, 64, 64, 1) == 0


def test_gated_arguments():
    lib = _lib.load_layers()

    def fwd(x=P, wg=P, wu=P, bg=None, bu=None, dtype=0, M=200, D=33, F=64, act=2, d=None, h=P,
            work=P, nbytes=1 << 40):
        return lib.ppo_layer_gated_forward(x, wg, wu, bg, bu, dtype, M, D, F, act, d, h, None,
                                           work, nbytes, None)

    assert fwd(dtype=3) == 1 and fwd(M=-1) == 1 and fwd(D=0) == 1 and fwd(F=0) == 1
    assert fwd(act=-1) == 1 and fwd(act=4) == 1 and fwd(d=drop(2.0)) == 1
    assert fwd(bg=P) == 1 and fwd(bu=P) == 1
    assert fwd(x=None) == 1 and fwd(wg=None) == 1 and fwd(wu=None) == 1 and fwd(h=None) == 1
    assert fwd(M=0, x=None, wg=None, wu=None, h=None) == 0
    assert fwd(M=1 << 28) == 3 and fwd(D=1 << 22) == 3
    need = lib.ppo_layer_gated_workspace_bytes(0, 200, 33, 64)
    assert need > 0 and fwd(nbytes=need - 1) == 2 and fwd(work=None) == 2
    assert lib.ppo_layer_gated_workspace_bytes(0, 0, 33, 64) == 0

    def bwd(dh=P, x=P, wg=P, wu=P, saved=P, dtype=0, M=200, D=33, F=64, act=2, d=None, dx=P,
            dwg=P, dwu=P, dbg=None, dbu=None, work=P, nbytes=1 << 40):
        return lib.ppo_layer_gated_backward(dh, x, wg, wu, saved, dtype, M, D, F, act, d, dx, dwg,
                                            dwu, dbg, dbu, work, nbytes, None)

    assert bwd(dtype=3) == 1 and bwd(M=0) == 1 and bwd(D=0) == 1 and bwd(F=-2) == 1
    assert bwd(act=7) == 1 and bwd(d=drop(-1.0)) == 1
    assert bwd(dwu=None) == 1 and bwd(dwg=None) == 1 and bwd(dbg=P) == 1 and bwd(dbu=P) == 1
    assert bwd(dh=None) == 1 and bwd(saved=None) == 1 and bwd(x=None) == 1 and bwd(wu=None) == 1
    need = lib.ppo_layer_gated_backward_workspace_bytes(0, 200, 33, 64)
    assert need > 0 and bwd(nbytes=need - 1) == 2 and bwd(work=None) == 2
    assert bwd(work=ctypes.c_void_p(4097)) == 2


def test_sizes_that_no_launch_holds():
    lib = _lib.load_layers()
    bytes_of = lib.ppo_layer_gated_workspace_bytes
    back = lib.ppo_layer_gated_backward_workspace_bytes
    eight = lib.ppo_layer_int8_linear_workspace_bytes
    # the largest that are documented have a plan, twice as large ones none
    assert bytes_of(0, 1 << 26, 8, 33) > 0 and back(0, 1 << 26, 8, 256) > 0
    assert bytes_of(0, 65, 3, 1 << 26) > 0 and eight(1 << 26, 256, 8, 1) > 0
    assert eight(65, 1 << 26, 7, 1) > 0
    for M, D, F in ((1 << 28, 8, 33), (64, 8, 1 << 28), (1 << 26, 8, 1 << 10), (1 << 27, 8, 513)):
        assert bytes_of(0, M, D, F) == 0 and back(0, M, D, F) == 0
    assert eight(1 << 28, 8, 8, 1) == 0 and eight(8, 1 << 28, 8, 1) == 0
    assert eight(1 << 26, 1 << 10, 8, 1) == 0


def test_saved_alignment():
    lib = _lib.load_layers()
    odd = ctypes.c_void_p(4104)
    assert lib.ppo_layer_gated_forward(P, P, P, None, None, 0, 4, 8, 8, 0, None, P, odd, P, 1 << 40,
                                       None) == 1
    assert lib.ppo_layer_gated_backward(P, P, P, P, odd, 0, 4, 8, 8, 0, None, P, P, P, None, None,
                                        P, 1 << 40, None) == 1


def test_workspaces_of_aligned_operands():
    """No room for copies of operands that need none."""
    lib, on = _lib.load_layers(), _lib.PPO_LAYER_ALIGNED
    fwd, bwd = lib.ppo_layer_gated_workspace_bytes, lib.ppo_layer_gated_backward_workspace_bytes
    eight = lib.ppo_layer_int8_linear_workspace_bytes
    M, D, F = 8192, 4096, 8192
    copies = 2 * (M * D + 2 * F * D)
    assert fwd(1, M, D, F) >= copies and fwd(1 | on, M, D, F) == 0
    dgu = 2 * 2 * M * F
    assert bwd(1, M, D, F) >= dgu + copies
    # (and the biases' sums and joins: 4 bytes of 2 F for every 16 rows)
    assert dgu <= bwd(1 | on, M, D, F) <= dgu + M // 16 * 2 * F * 4
    assert eight(M, F, D, 0) >= M * D + F * D and eight(M, F, D, on) == 0
    assert eight(M, F, D, 1) >= M * D + F * D
    assert M * D <= eight(M, F, D, 1 | on) <= M * D + 4 * M + 512
    # rows that are no multiple of 16 bytes need their copies at any address
    for d in (4095, 4097):
        assert fwd(1 | on, M, d, F) == fwd(1, M, d, F) > 0
        assert bwd(1 | on, M, d, F) == bwd(1, M, d, F)
        assert eight(M, F, d, on) == eight(M, F, d, 0) > 0
    # a promise that does not hold, and less than was asked for
    odd = ctypes.c_void_p(4104)

    def gated(x=P, wg=P, wu=P, dtype=on, M=200, D=32, F=64, work=P, nbytes=1 << 40):
        return (lib.ppo_layer_gated_forward(x, wg, wu, None, None, dtype, M, D + 1, F, 0, None, P,
                                            None, work, nbytes, None),
                lib.ppo_layer_gated_backward(P, x, wg, wu, P, dtype, M, D, F, 0, None, P, P, P,
                                             None, None, work, nbytes, None))

    for kw in (dict(x=odd), dict(wg=odd), dict(wu=odd), dict(dtype=3 | on), dict(dtype=-1)):
        assert gated(**kw) == (1, 1)
    assert gated(nbytes=min(fwd(on, 200, 33, 64), bwd(on, 200, 32, 64)) - 1) == (2, 2)
    f = lib.ppo_layer_int8_linear
    assert f(None, odd, P, P, P, None, on, 200, 64, 64, P, P, 1 << 40, None) == 1
    assert f(P, None, None, odd, P, None, on, 200, 64, 64, P, P, 1 << 40, None) == 1
    need = eight(200, 64, 64, 1 | on)
    assert f(P, None, None, P, P, None, on, 200, 64, 64, P, P, need - 1, None) == 2
    # at any address as before
    assert f(P, None, None, P, P, None, 0, 200, 64, 64, P, P, eight(200, 64, 64, 1) - 1, None) == 2


def test_cpu_tensors_and_types_are_refused():
    x, w = torch.zeros(4, 8), torch.zeros(6, 8)
    for call in (lambda: ppo_amd.dropout(x, 0.1, 1), lambda: ppo_amd.gated_ffn(x, w, w),
                 lambda: ppo_amd.quantize_rows(x),
                 lambda: ppo_amd.int8_linear(x, w.to(torch.int8), torch.ones(6))):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()
    with pytest.raises(TypeError):
        ppo_amd.dropout([1.0], 0.1, 1)


SCHEMAS = {
    "dropout": "ppo_amd::dropout(Tensor x, float p, SymInt seed, Tensor? seed_at, Tensor? rows) "
               "-> Tensor",
    "gated_ffn": "ppo_amd::gated_ffn(Tensor x, Tensor w_gate, Tensor w_up, Tensor? b_gate, "
                 "Tensor? b_up, str activation, float dropout_p, SymInt seed, Tensor? seed_at, "
                 "Tensor? rows) -> (Tensor, Tensor)",
    "quantize_rows": "ppo_amd::quantize_rows(Tensor x) -> (Tensor, Tensor)",
    "int8_linear": "ppo_amd::int8_linear(Tensor x, Tensor weight, Tensor weight_scale, "
                   "Tensor? bias, Tensor? x_scale, ScalarType? out_dtype) -> Tensor",
}


@pytest.mark.parametrize("name", sorted(SCHEMAS))
def test_operator_schema(name):
    assert str(getattr(torch.ops.ppo_amd, name).default._schema) == SCHEMAS[name]


def test_operators_fake_shapes_and_cpu():
    from torch._subclasses.fake_tensor import FakeTensorMode

    op = torch.ops.ppo_amd
    with FakeTensorMode():
        x, w, b = (torch.empty(s, device="cuda", dtype=torch.bfloat16)
                   for s in ((3, 5, 8), (7, 8), (7,)))
        assert op.dropout(x, 0.1, 1, None, None).shape == (3, 5, 8)
        h, saved = op.gated_ffn(x, w, w, b, b, "silu", 0.1, 1, None, None)
        assert h.shape == (3, 5, 7) and h.dtype == torch.bfloat16
        assert saved.shape == (2, 15, 8) and saved.dtype == torch.float32
        grads = op.gated_ffn_backward(h, x, w, w, saved, True, "silu", 0.1, 1, None, None)
        assert [g.shape for g in grads] == [(3, 5, 8), (7, 8), (7, 8), (7,), (7,)]
        q, s = op.quantize_rows(w)
        assert q.shape == (7, 8) and q.dtype == torch.int8 and s.shape == (7,)
        assert op.int8_linear(x, q, s, None, None, None).shape == (3, 5, 7)
    with pytest.raises(NotImplementedError):
        op.dropout(torch.zeros(2, 2), 0.1, 1, None, None)


def _backward_faults(torch_device="cuda"):
    """(arguments of a gated backward, the error) with one of them wrong, as
    fake tensors: nothing may be launched on them."""
    bf = torch.bfloat16

    def e(*shape, dtype=bf, device=torch_device):
        return torch.empty(shape, dtype=dtype, device=device)

    def args(**kw):
        a = dict(dh=e(3, 5, 7), x=e(3, 5, 8), wg=e(7, 8), wu=e(7, 8),
                 saved=e(2, 15, 8, dtype=torch.float32), seed_at=None, rows=None)
        a.update(kw)
        return a

    i64 = dict(dtype=torch.int64)
    return [(args(dh=e(2, 5, 7)), ValueError), (args(dh=e(15, 6)), ValueError),
            (args(dh=e(3, 7, 5).transpose(1, 2)), ValueError),
            (args(dh=e(3, 5, 7, dtype=torch.float16)), TypeError),
            (args(dh=e(3, 5, 7, device="cpu")), RuntimeError),
            (args(saved=e(2, 15, 7, dtype=torch.float32)), ValueError),
            (args(saved=e(2, 14, 8, dtype=torch.float32)), ValueError),
            (args(saved=e(2, 15, 8)), TypeError),
            (args(saved=e(2, 15, 8, dtype=torch.float32, device="cpu")), RuntimeError),
            (args(wu=e(6, 8)), ValueError), (args(wg=e(7, 9), wu=e(7, 9)), ValueError),
            (args(wg=e(7, 8, dtype=torch.float32)), TypeError), (args(x=e(3, 4, 8)), ValueError),
            (args(rows=e(14, **i64)), ValueError), (args(rows=e(15, dtype=torch.int32)), TypeError),
            (args(rows=e(15, device="cpu", **i64)), RuntimeError),
            (args(seed_at=e(2, **i64)), ValueError),
            (args(seed_at=e(1, device="cpu", **i64)), RuntimeError)]


def test_backward_operator_refuses():
    """ppo_amd::gated_ffn_backward checks what it hands to the kernels."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    from ppo_amd import torch_ops

    f = torch_ops.gated_ffn_backward._init_fn
    with FakeTensorMode():
        for a, error in _backward_faults():
            with pytest.raises(error, match="must|dtype|expected|no CPU fallback"):
                f(a["dh"], a["x"], a["wg"], a["wu"], a["saved"], False, "silu", 0.1, 1,
                  a["seed_at"], a["rows"])
        with pytest.raises(ValueError, match="activation"):
            f(a["dh"], a["x"], a["wg"], a["wu"], a["saved"], False, "swish", 0.1, 1, None, None)
        with pytest.raises(ValueError, match="probability"):
            f(a["dh"], a["x"], a["wg"], a["wu"], a["saved"], False, "silu", 1.5, 1, None, None)


def test_backward_nodes_refuse_what_hooks_hand_back():
    """The Python autograd functions check their saved tensors before a launch."""
    from types import SimpleNamespace

    from torch._subclasses.fake_tensor import FakeTensorMode

    def ctx(*saved):
        return SimpleNamespace(p=0.1, act=2, seed=None if saved[-2] is not None else 1,
                               saved_tensors=saved, needs_input_grad=(True,) * 5)

    with FakeTensorMode(), torch.no_grad():
        for a, error in _backward_faults():
            with pytest.raises(error, match="must|dtype|expected|no CPU fallback"):
                dh = a["dh"].contiguous()  # (the node makes it so)
                if not a["dh"].is_contiguous():
                    raise ValueError("must be contiguous")
                layers._GatedFFN.backward(ctx(a["x"], a["wg"], a["wu"], a["saved"], a["seed_at"],
                                              a["rows"]), dh)
            if a["seed_at"] is not None or a["rows"] is not None:
                with pytest.raises(error, match="must|dtype|expected|no CPU fallback"):
                    layers._Dropout.backward(ctx(a["seed_at"], a["rows"]), a["dh"])


def test_module_arguments():
    with pytest.raises(ValueError):
        ppo_amd.GatedLinear(4, 4, activation="swish")
    with pytest.raises(ValueError):
        ppo_amd.GatedLinear(4, 4, dropout=1.5)
    m = ppo_amd.GatedMLP(6, 16, 3, dropout=0.1, seed=5)
    assert [tuple(p.shape) for p in m.parameters()] == [
        (16, 6), (16,), (16, 6), (16,), (16, 16), (16,), (16, 16), (16,), (3, 16), (3,)]
    assert [int(l.seed) for l in m.hidden] == [10, 11]
    m.reseed(7)
    assert [int(l.seed) for l in m.hidden] == [14, 15]
    assert layers.ACTIVATIONS.keys() == {"relu", "tanh", "silu", "gelu"}


def test_module_seeds_of_any_size():
    """A module's seed is the low 64 bits of an int, as the functions' is."""
    m = ppo_amd.GatedMLP(6, 16, 3, dropout=0.1, seed=2**62)
    assert [int(l.seed) for l in m.hidden] == [-2**63, -2**63 + 1]
    m.reseed(2**64 - 1)
    assert [int(l.seed) for l in m.hidden] == [-2, -1]
    layer = ppo_amd.GatedLinear(4, 4, seed=2**64 - 1)
    assert int(layer.seed) == -1
    layer.reseed(-2**63 - 1)
    assert int(layer.seed) == 2**63 - 1
    layer.reseed(np.int64(7))
    assert int(layer.seed) == 7 and int(ppo_amd.GatedLinear(4, 4, seed=np.int32(-2)).seed) == -2


# --- the oracle -------------------------------------------------------------------------

def test_philox_known_answers():
    """Vectors published with the generator's paper: counter and key all
    zeros, all ones, for 7 and 10 rounds."""
    zero, ones = [np.uint64(0)] * 4, [np.uint64(0xFFFFFFFF)] * 4
    hexes = lambda words: " ".join(f"{int(w):08x}" for w in words)  # noqa: E731
    assert hexes(ref.philox4x32(zero, (0, 0), 7)) == "5f6fb709 0d893f64 4f121f81 4f730a48"
    assert hexes(ref.philox4x32(zero, (0, 0), 10)) == "6627e8d5 e169c58d bc57ac4c 9b00dbd8"
    assert hexes(ref.philox4x32(ones, (0xFFFFFFFF, 0xFFFFFFFF), 10)) == \
        "408f276d 41c83b0e a20bc7c6 6d5451fd"


def test_keep_mask_statistics():
    n = 1 << 20
    for p in (0.1, 0.5):
        keep = ref.keep_mask(p, 1234567890123, np.arange(1024), 1024)
        assert abs(keep.mean() - (1 - p)) < 5 * np.sqrt(p * (1 - p) / n)
    assert ref.keep_mask(0.0, 9, [3], 40).all() and not ref.keep_mask(1.0, 9, [3], 40).any()
    # a row's mask goes by its id alone
    a, b = ref.keep_mask(0.5, 7, [5, 1 << 33, 2], 37), ref.keep_mask(0.5, 7, [1 << 33], 50)
    assert (a[1] == b[0, :37]).all() and (a[0] != a[2]).any()


@pytest.mark.parametrize("act", ["relu", "tanh", "silu", "gelu"])
def test_oracle_gradients_are_autograds(act):
    g = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    x, wg, wu, bg, bu, dh = r(7, 5), r(6, 5), r(6, 5), r(6), r(6), r(7, 6)
    keep = torch.rand(7, 6, generator=g) < 0.7
    leaves = [t.clone().requires_grad_() for t in (x, wg, wu, bg, bu)]
    f = {"relu": torch.relu, "tanh": torch.tanh, "silu": torch.nn.functional.silu,
         "gelu": torch.nn.functional.gelu}[act]
    lx, lwg, lwu, lbg, lbu = leaves
    h = f(lx @ lwg.T + lbg) * (lx @ lwu.T + lbu) * keep / 0.7
    h.backward(dh)
    want, gg, uu = ref.gated_ffn(x, wg, wu, bg, bu, act, keep, 0.3)
    torch.testing.assert_close(want, h.detach(), rtol=1e-12, atol=1e-12)
    got = ref.gated_ffn_grads(x, wg, wu, gg, uu, act, dh, keep, 0.3)
    for a, leaf in zip(got, leaves):
        torch.testing.assert_close(a, leaf.grad, rtol=1e-11, atol=1e-12)


def test_oracle_quantize():
    x = np.array([[127.0, -63.5, 0.5, 1.5], [0, 0, 0, 0], [1, np.inf, 0, 0], [np.nan, 1, 2, 3]],
                 dtype=np.float32)
    q, s = ref.quantize_rows(x)
    assert s[0] == 1 and s[1] == 0 and np.isnan(s[2:]).all()
    assert q.tolist() == [[127, -64, 0, 2], [0] * 4, [0] * 4, [0] * 4]
