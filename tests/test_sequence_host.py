"""Token-sequence operators without a GPU: the oracle's gradients against differences, the refusals of the Python
layer (on tensors that only pretend to sit on a GPU) and of the C entry points."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import sequence_oracle as so
from superresolution_amd import _lib, sequence


# ---- the oracle ------------------------------------------------------------------------------------------------
def _leaf(g, *shape, lo=None):
    t = torch.randn(*shape, generator=g, dtype=torch.float64)
    return (t if lo is None else lo * (0.5 + torch.rand(*shape, generator=g, dtype=torch.float64))).requires_grad_(True)


def _check_grads(names, tensors, forward, grads):
    """Central differences of the oracle's forward pass along every input, against its gradient formulas."""
    for name, t in zip(names, tensors):
        v = torch.randn(t.shape, generator=torch.Generator().manual_seed(7), dtype=torch.float64)
        d = 1e-6
        with torch.no_grad():
            t += d * v
            up = forward()
            t -= 2 * d * v
            down = forward()
            t += d * v
        slope, formula = float(up - down) / (2 * d), float((grads[name] * v).sum())
        assert abs(slope - formula) <= 1e-6 * max(1.0, abs(formula)), (name, slope, formula)


@pytest.mark.parametrize("bias", [True, False])
def test_oracle_norm_gradient(bias):
    g = torch.Generator().manual_seed(0)
    x, w, b, dy = _leaf(g, 4, 7), _leaf(g, 7), _leaf(g, 7) if bias else None, _leaf(g, 4, 7).detach()
    grads = so.norm(x.detach(), w.detach(), None if b is None else b.detach(), 1e-5, dy)[0]
    names, ts = ["dx", "dw"] + ["db"] * bias, [x, w] + [b] * bias
    _check_grads(names, ts, lambda: (so.norm(x, w, b, 1e-5)[0]["y"] * dy).sum(), grads)


@pytest.mark.parametrize("L", [1, 2, 9])
def test_oracle_conv_gradient(L):
    g = torch.Generator().manual_seed(1)
    x, w, b, h = _leaf(g, 2, 3, L), _leaf(g, 3, 4), _leaf(g, 3), _leaf(g, 2, 3, 3)
    dy, dend = _leaf(g, 2, 3, L).detach(), _leaf(g, 2, 3, 3).detach()

    def loss():
        o = so.conv(x, w, b, h, True)[0]
        return (o["y"] * dy).sum() + (o["end"] * dend).sum()
    grads = so.conv(x.detach(), w.detach(), b.detach(), h.detach(), True, dy, dend)[0]
    _check_grads(["dx", "dw", "db", "dstate"], [x, w, b, h], loss, grads)


@pytest.mark.parametrize("softplus", [True, False])
def test_oracle_scan_gradient(softplus):
    g = torch.Generator().manual_seed(2)
    x, B, C, z, D = _leaf(g, 2, 4, 6), _leaf(g, 2, 2, 3, 6), _leaf(g, 2, 2, 3, 6), _leaf(g, 2, 4, 6), _leaf(g, 4)
    delta, A, bias, h0 = _leaf(g, 2, 4, 6, lo=0.3), _leaf(g, 4, 3, lo=-1.0), _leaf(g, 4, lo=0.1), _leaf(g, 2, 4, 3)
    dy, dlast = _leaf(g, 2, 4, 6).detach(), _leaf(g, 2, 4, 3).detach()

    def loss():
        o = so.scan(x, delta, A, B, C, D, z, bias, softplus, h0)[0]
        return (o["y"] * dy).sum() + (o["last"] * dlast).sum()
    ts = [x, delta, A, B, C, D, z, bias, h0]
    grads = so.scan(*[t.detach() for t in ts[:8]], softplus, h0.detach(), dy, dlast)[0]
    _check_grads(["dx", "ddelta", "dA", "dB", "dC", "dD", "dz", "ddelta_bias", "dh0"], ts, loss, grads)


# ---- refusals of the Python layer -------------------------------------------------------------------------------
@pytest.fixture
def fake():
    with FakeTensorMode(allow_non_fake_inputs=True):
        yield lambda *shape, dtype=torch.float32: torch.empty(*shape, dtype=dtype, device="cuda:0")


def test_cpu_tensors_are_refused():
    t = torch.zeros
    for call in (lambda: sequence.layernorm(t(2, 3), t(3)), lambda: sequence.causal_conv1d(t(1, 2, 3), t(2, 4)),
                 lambda: sequence.causal_conv1d_update(t(1, 2), t(1, 2, 3), t(2, 4)),
                 lambda: sequence.selective_scan(t(1, 2, 3), t(1, 2, 3), t(2, 4), t(1, 1, 4, 3), t(1, 1, 4, 3)),
                 lambda: sequence.selective_scan_update(t(1, 2, 4), t(1, 2), t(1, 2), t(2, 4), t(1, 1, 4), t(1, 1, 4))):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


def test_layernorm_refuses(fake):
    n = sequence.layernorm
    with pytest.raises(RuntimeError, match="dtype"):
        n(fake(2, 8, dtype=torch.float16), fake(8))
    with pytest.raises(RuntimeError, match="weight: dtype"):
        n(fake(2, 8), fake(8, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="last dimension"):
        n(fake(2, 8193), fake(8193))
    with pytest.raises(RuntimeError, match="last dimension"):
        n(fake(2, 0), fake(0))
    with pytest.raises(RuntimeError, match="weight: shape"):
        n(fake(2, 8), fake(7))
    with pytest.raises(RuntimeError, match="bias: shape"):
        n(fake(2, 8), fake(8), fake(8, 1))
    with pytest.raises(RuntimeError, match="eps"):
        n(fake(2, 8), fake(8), eps=-1e-5)
    with pytest.raises(RuntimeError, match="eps"):
        n(fake(2, 8), fake(8), eps=float("nan"))
    with pytest.raises(RuntimeError, match="weight: tensor is on cpu"):
        n(fake(2, 8), torch.zeros(8))


def test_conv_refuses(fake):
    c, x = sequence.causal_conv1d, fake(2, 6, 10)
    for w in ((6, 1), (6, 5), (5, 4), (6, 2, 4)):
        with pytest.raises(RuntimeError, match="weight"):
            c(x, fake(*w))
    with pytest.raises(RuntimeError, match="activation"):
        c(x, fake(6, 4), activation="gelu")
    with pytest.raises(RuntimeError, match="initial_state: shape"):
        c(x, fake(6, 4), initial_state=fake(2, 6, 4))
    with pytest.raises(RuntimeError, match="initial_state"):
        c(x, fake(6, 4), initial_state=fake(2, 6, 3, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="batch, channel, token"):
        c(fake(6, 10), fake(6, 4))
    u, x1 = sequence.causal_conv1d_update, fake(2, 6)
    with pytest.raises(RuntimeError, match="state: shape"):
        u(x1, fake(2, 6, 4), fake(6, 4))
    with pytest.raises(RuntimeError, match="contiguous"):
        u(x1, fake(2, 3, 6).transpose(1, 2), fake(6, 4))
    with pytest.raises(RuntimeError, match="state_out"):
        u(x1, fake(2, 6, 3), fake(6, 4), state_out=fake(2, 6, 3, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="inference only"):
        u(x1, fake(2, 6, 3), fake(6, 4).requires_grad_(True))


def test_scan_refuses(fake):
    s, x, A, B = sequence.selective_scan, fake(2, 6, 10), fake(6, 8), fake(2, 1, 8, 10)
    with pytest.raises(RuntimeError, match="A "):
        s(x, x, fake(6, 33), B, B)
    with pytest.raises(RuntimeError, match="A "):
        s(x, x, fake(5, 8), B, B)
    with pytest.raises(RuntimeError, match="groups"):
        s(x, x, A, fake(2, 4, 8, 10), fake(2, 4, 8, 10))
    with pytest.raises(RuntimeError, match="B: shape"):
        s(x, x, A, fake(2, 1, 8, 9), B)
    with pytest.raises(RuntimeError, match="C: shape"):
        s(x, x, A, B, fake(2, 2, 8, 10))
    with pytest.raises(RuntimeError, match="delta: shape"):
        s(x, fake(2, 6, 1), A, B, B)
    with pytest.raises(RuntimeError, match="z: shape"):
        s(x, x, A, B, B, z=fake(2, 6, 9))
    with pytest.raises(RuntimeError, match="D: shape"):
        s(x, x, A, B, B, fake(6, 1))
    with pytest.raises(RuntimeError, match="delta_bias: shape"):
        s(x, x, A, B, B, delta_bias=fake(1))
    with pytest.raises(RuntimeError, match="initial_state: shape"):
        s(x, x, A, B, B, initial_state=fake(2, 6, 10))
    with pytest.raises(RuntimeError, match="initial_state: dtype"):
        s(x, x, A, B, B, initial_state=fake(2, 6, 8, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="delta"):
        s(x, fake(2, 6, 10, dtype=torch.bfloat16), A, B, B)
    u, x1, B1 = sequence.selective_scan_update, fake(2, 6), fake(2, 1, 8)
    with pytest.raises(RuntimeError, match="state: shape"):
        u(fake(2, 8, 6), x1, x1, A, B1, B1)
    with pytest.raises(RuntimeError, match="state.*dtype"):
        u(fake(2, 6, 8, dtype=torch.bfloat16), x1, x1, A, B1, B1)
    with pytest.raises(RuntimeError, match="contiguous"):
        u(fake(2, 8, 6).transpose(1, 2), x1, x1, A, B1, B1)
    with pytest.raises(RuntimeError, match="inference only"):
        u(fake(2, 6, 8), x1, x1, A.requires_grad_(True), B1, B1)


# ---- refusals of the C entry points (nothing is launched) -----------------------------------------------------------
def test_c_entry_points_refuse():
    lib = _lib.load()
    err = lambda: lib.rst_last_error().decode()
    p = 4096                                                              # never read: the arguments are refused first
    assert lib.rst_rows_norm_fwd(None, 0, p, None, p, 4, 8, 1e-5, None) == 1 and "null" in err()
    assert lib.rst_rows_norm_fwd(p, 2, p, None, p, 4, 8, 1e-5, None) == 1 and "dtype" in err()
    assert lib.rst_rows_norm_fwd(p, 0, p, None, p, 0, 8, 1e-5, None) == 1 and "empty" in err()
    assert lib.rst_rows_norm_fwd(p, 0, p, None, p, 4, 8193, 1e-5, None) == 1 and "8192" in err()
    assert lib.rst_rows_norm_fwd(p, 0, p, None, p, 4, 8, float("nan"), None) == 1 and "eps" in err()
    need = lib.rst_rows_norm_bwd_workspace_bytes(4, 8)
    assert need > 0 and lib.rst_rows_norm_bwd_workspace_bytes(0, 8) == 0
    assert lib.rst_rows_norm_bwd(p, 0, p, 1, p, p, p, None, 4, 8, 1e-5, p, need, None) == 1 and "dbias" in err()
    assert lib.rst_rows_norm_bwd(p, 0, p, 0, p, p, p, None, 4, 8, 1e-5, p, need - 1, None) == 3 and "too small" in err()
    assert lib.rst_causal_conv1d_fwd(p, 0, p, None, None, p, None, 1, 2, 8, 5, 0, None) == 1 and "width" in err()
    assert lib.rst_causal_conv1d_fwd(p, 0, p, None, None, p, None, 1, 2, 0, 4, 0, None) == 1 and "empty" in err()
    need = lib.rst_causal_conv1d_bwd_workspace_bytes(1, 2, 100)
    assert lib.rst_causal_conv1d_bwd(p, 0, p, None, None, p, None, p, p, None, None, 1, 2, 100, 4, 0, p, need - 1, None) == 3
    assert lib.rst_causal_conv1d_update(p, 0, None, p, p, None, p, 1, 2, 4, 0, None) == 1 and "null" in err()

    def desc(B=1, D=4, G=1, N=8, L=10, dtype=0):
        return ctypes.byref(_lib.ScanDesc(B, D, G, N, L, dtype, 1))
    ins = _lib.ScanInputs(p, p, p, p, p, None, None, None)
    for kw in (dict(B=0), dict(D=0), dict(L=0), dict(N=0), dict(N=33), dict(G=3), dict(G=0), dict(dtype=7), dict(B=70000), dict(L=(1 << 24) + 1)):
        assert lib.rst_scan_saved_bytes(desc(**kw)) == 0 and lib.rst_scan_bwd_workspace_bytes(desc(**kw)) == 0
        assert lib.rst_scan_fwd(desc(**kw), ctypes.byref(ins), None, p, None, None, p, 1 << 40, None) == 1, kw
    assert lib.rst_scan_workspace_bytes(desc()) == 0                      # one chunk: no scratch
    need = lib.rst_scan_workspace_bytes(desc(L=5000))
    assert need > 0
    assert lib.rst_scan_fwd(desc(L=5000), ctypes.byref(ins), None, p, None, None, p, need - 1, None) == 3
    assert lib.rst_scan_fwd(desc(L=5000), ctypes.byref(ins), None, p, None, None, None, need, None) == 3
    assert lib.rst_scan_fwd(desc(L=5000), ctypes.byref(ins), None, p, None, None, p + 4, need, None) == 1 and "aligned" in err()
    assert lib.rst_scan_fwd(desc(), ctypes.byref(_lib.ScanInputs(p, p, p, p, None, None, None, None)), None, p, None, None, p, need, None) == 1
    outs = _lib.ScanGrads(p, p, p, p, p, None, None, None)
    need = lib.rst_scan_bwd_workspace_bytes(desc())
    gated = _lib.ScanInputs(p, p, p, p, p, None, p, None)
    assert lib.rst_scan_bwd(desc(), ctypes.byref(gated), p, p, None, ctypes.byref(outs), None, p, need, None) == 1 and "gradient" in err()
    assert lib.rst_scan_bwd(desc(), ctypes.byref(ins), None, p, None, ctypes.byref(outs), None, p, need, None) == 1 and "null" in err()
    assert lib.rst_scan_update(desc(), ctypes.byref(ins), p, p, p, None) == 1 and "one token" in err()
    assert ctypes.sizeof(_lib.ScanDesc) == 32 and ctypes.sizeof(_lib.ScanInputs) == 64


def test_the_longest_row(fake):
    with pytest.raises(RuntimeError, match="at most 16777216"):
        sequence.selective_scan(fake(1, 2, (1 << 24) + 1), fake(1, 2, (1 << 24) + 1), fake(2, 1), fake(1, 1, 1, (1 << 24) + 1),
                                fake(1, 1, 1, (1 << 24) + 1))


# ---- forward-mode derivatives: there are none, and none is dropped ---------------------------------------------------
def _dual_calls(make):
    """Each entry point with every one of its tensors in turn, as (name, call of that tensor's dual)."""
    x, w = make(2, 6, 10), make(6, 4)
    x1, w1, s1 = make(2, 6), make(6, 4), make(2, 6, 3)
    A, B, B1, v, h = make(6, 8), make(2, 1, 8, 10), make(2, 1, 8), make(6), make(2, 6, 8)
    sq = sequence
    table = [(lambda x, w, b: sq.layernorm(x, w, b), [make(2, 8), make(8), make(8)]),
             (lambda x, w, b, h: sq.causal_conv1d(x, w, b, initial_state=h, activation="silu"), [x, w, v, s1]),
             (lambda x, s, w, b, o: sq.causal_conv1d_update(x, s, w, b, state_out=o), [x1, s1, w1, v, make(2, 6, 3)]),
             (lambda x, d, A, B, C, D, z, b, h: sq.selective_scan(x, d, A, B, C, D, z=z, delta_bias=b, initial_state=h),
              [x, x, A, B, B, v, x, v, h]),
             (lambda s, x, d, A, B, C, D, z, b, o: sq.selective_scan_update(s, x, d, A, B, C, D, z=z, delta_bias=b, state_out=o),
              [h, x1, x1, A, B1, B1, v, x1, v, make(2, 6, 8)])]
    for call, tensors in table:
        for i, t in enumerate(tensors):
            yield lambda dual, call=call, tensors=tensors, i=i: call(*tensors[:i], dual, *tensors[i + 1:]), t


@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_tangents_are_refused(fake, monkeypatch, grad):
    """A dual tensor has requires_grad == False: it must not take the way without gradients, whose result has no tangent."""
    monkeypatch.setattr(sequence, "_call", lambda name, *args: pytest.fail(f"{name} was launched"))
    fw = torch.autograd.forward_ad
    n = 0
    for call, t in _dual_calls(fake):
        with fw.dual_level(), torch.set_grad_enabled(grad):
            with pytest.raises(NotImplementedError):
                call(fw.make_dual(t, torch.ones_like(t)))
        n += 1
    assert n == 31


def test_update_does_not_write_into_a_leaf(fake):
    """`state_out` with a gradient of its own: torch refuses an in-place write to such a tensor, and so does an update."""
    with pytest.raises(RuntimeError, match="inference only"):
        sequence.causal_conv1d_update(fake(2, 6), fake(2, 6, 3), fake(6, 4), state_out=fake(2, 6, 3).requires_grad_(True))
    with pytest.raises(RuntimeError, match="inference only"):
        sequence.selective_scan_update(fake(2, 6, 8), fake(2, 6), fake(2, 6), fake(6, 8), fake(2, 1, 8), fake(2, 1, 8),
                                       state_out=fake(2, 6, 8).requires_grad_(True))


# ---- what an update writes to is known to autograd --------------------------------------------------------------------
def test_updates_move_the_version_counter(fake, monkeypatch):
    """The state is written through its address: the tensor's version moves as with any in-place operation of torch, the
    state's own only where it is what is written."""
    calls = []
    monkeypatch.setattr(sequence, "_call", lambda name, *args: calls.append(name))
    conv = lambda s, **kw: sequence.causal_conv1d_update(fake(2, 6), s, fake(6, 4), **kw)
    scan = lambda s, **kw: sequence.selective_scan_update(s, fake(2, 6), fake(2, 6), fake(6, 8), fake(2, 1, 8), fake(2, 1, 8), **kw)
    for update, shape in ((conv, (2, 6, 3)), (scan, (2, 6, 8))):
        s, o = fake(*shape), fake(*shape)
        whole = fake(2, *shape)
        update(s)
        assert s._version == 1
        update(s, state_out=o)
        assert s._version == 1 and o._version == 1
        update(whole[1])                                                  # a view: the tensor it is a part of was written to
        assert whole._version == 1
        with torch.inference_mode():
            update(fake(*shape))
    assert len(calls) == 8
    empty = fake(0, 6, 3)
    sequence.causal_conv1d_update(fake(0, 6), empty, fake(6, 4))
    assert empty._version == 0 and len(calls) == 8


def test_workspace_sizes_of_shapes_out_of_range():
    """0 bytes, as for an empty shape, and the reason: a row of 2^35 tokens used to end the process in a division by zero."""
    lib = _lib.load()
    for B, D, L in ((1, 1, 1 << 35), (1, 1, (1 << 31) + 1), (1 << 16, 1 << 15, 8), (-1, 4, 8), (4, 4, -8)):
        assert lib.rst_causal_conv1d_bwd_workspace_bytes(B, D, L) == 0, (B, D, L)
        assert b"causal_conv1d_bwd_workspace_bytes" in lib.rst_last_error()
    assert lib.rst_causal_conv1d_bwd_workspace_bytes(1, 1, 1 << 31) > 0
    assert lib.rst_causal_conv1d_bwd_workspace_bytes(1 << 15, 1 << 15, 8) > 0


def test_norm_workspace_fits_the_rows():
    """A row of partial sums for every block that runs: at most 1024, and no more than there are rows."""
    size = _lib.load().rst_rows_norm_bwd_workspace_bytes
    assert size(1, 8192) == 8192 * 8 and size(64, 384) <= 64 * 384 * 8 and size(1 << 20, 96) == 1024 * 96 * 8
    for C in (1, 5, 24, 96, 181, 513, 1000, 2048, 4096, 8192):
        sizes = [size(rows, C) for rows in (1, 2, 7, 64, 1000, 1 << 20)]
        assert sizes == sorted(sizes) and sizes[0] == 8 * C and sizes[-1] == 1024 * 8 * C, C
