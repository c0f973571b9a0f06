"""Sequence operators without a GPU: the 64-bit oracle against itself in other forms, and every refusal."""
import ctypes as C

import numpy as np
import pytest
import torch

from oracle import sequence_numpy as sn

NS5 = [(3.4445, -4.7750, 2.0315)] * 5


def _problem(rng, B=2, T=7, G=1, H=2, K=3, V=4, per_token=True):
    q, k = rng.standard_normal((2, B, T, G, K))
    v = rng.standard_normal((B, T, H, V))
    g = -rng.random((B, T, H)) if per_token else -rng.random(H)
    return q, k, v, g, rng.standard_normal((B, H, K, V))


def test_the_recurrence_is_its_quadratic_form():
    """o_i = s sum_{j<=i} exp(G_i - G_j) (q_i.k_j) v_j + s exp(G_i) S_0' q_i."""
    rng = np.random.default_rng(0)
    q, k, v, g, s0 = _problem(rng)
    o, _ = sn.attention(q, k, v, g, 0.7, s0)
    for b in range(2):
        for h in range(2):
            cum = np.cumsum(g[b, :, h])
            D = np.exp(np.tril(cum[:, None] - cum[None, :])) * np.tri(7)
            want = 0.7 * (((q[b, :, 0] @ k[b, :, 0].T) * D) @ v[b, :, h] + np.exp(cum)[:, None] * (q[b, :, 0] @ s0[b, h]))
            np.testing.assert_allclose(o[b, :, h], want, rtol=1e-12, atol=1e-12)


@pytest.mark.parametrize("per_token", [True, False])
@pytest.mark.parametrize("lengths", [None, [7, 0], [3, 5]])
def test_the_oracles_gradient_against_differences(per_token, lengths):
    rng = np.random.default_rng(1)
    q, k, v, g, s0 = _problem(rng, per_token=per_token)
    go, gs = rng.standard_normal(v.shape), rng.standard_normal(s0.shape)
    grad = sn.attention_gradient(q, k, v, g, go, 0.7, s0, lengths, gs)

    def loss(**kw):
        x = dict(q=q, k=k, v=v, log_decay=g, initial_state=s0) | kw
        o, S = sn.attention(x["q"], x["k"], x["v"], x["log_decay"], 0.7, x["initial_state"], lengths)
        return np.sum(o * go) + np.sum(S * gs)

    for name, x in dict(q=q, k=k, v=v, log_decay=g, initial_state=s0).items():
        step = 1e-5 * rng.standard_normal(x.shape)
        want = loss(**{name: x + step}) - loss(**{name: x - step})
        # central differences: off by the third derivative, ~ |step|^3 times a few hundred
        assert abs(2 * np.sum(grad[name] * step) - want) < 1e-11 * max(1.0, abs(want) / 1e-5), name


@pytest.mark.parametrize("per_token", [True, False])
@pytest.mark.parametrize("lengths", [None, [7, 0], [3, 5]])
def test_the_batched_oracle_is_the_other(per_token, lengths):
    from oracle import sequence_torch as st

    rng = np.random.default_rng(5)
    q, k, v, g, s0 = _problem(rng, G=2, H=4, per_token=per_token)
    go, gs = rng.standard_normal(v.shape), rng.standard_normal(s0.shape)
    for first, last in ((s0, gs), (None, None)):
        for a, b in zip(sn.attention(q, k, v, g, 0.7, first, lengths), st.attention(q, k, v, g, 0.7, first, lengths)):
            np.testing.assert_allclose(a, b, rtol=1e-13, atol=1e-13)
        a, b = (m.attention_gradient(q, k, v, g, go, 0.7, first, lengths, last) for m in (sn, st))
        assert a.keys() == b.keys()
        for n in a:
            np.testing.assert_allclose(a[n], b[n], rtol=1e-12, atol=1e-12, err_msg=n)


def test_orthogonalise_maps_the_singular_values():
    rng = np.random.default_rng(2)
    for shape in ((5, 9), (9, 5), (6, 6)):
        M = rng.standard_normal(shape)
        U, S, Vh = np.linalg.svd(M, full_matrices=False)
        S = S / (np.linalg.norm(S) + 1e-7)
        for a, b, c in NS5:
            S = a * S + b * S ** 3 + c * S ** 5
        np.testing.assert_allclose(sn.orthogonalise(M, NS5), (U * S) @ Vh, atol=1e-12)


# ------------------------------------------------------------------------------------------------------- refusals, in C
@pytest.fixture
def lib():
    from pymc_statespace_amd import _lib

    return _lib.load()


@pytest.fixture
def handle():
    # a handle's memory without a device: every call below is refused before a device is touched
    return C.cast(C.create_string_buffer(1 << 16), C.c_void_p)


def _dims(**kw):
    from pymc_statespace_amd import _lib

    x = dict(B=1, T=4, G=1, H=2, K=8, V=8, dtype=1, decay_per_token=1, scale=1.0) | kw
    strides = {n: x.pop(n) for n in ("q_stride", "k_stride", "v_stride", "g_o_stride") if n in x}
    d = _lib.KfAttentionDims(**x)
    for n, s in strides.items():
        getattr(d, n)[:] = s
    return d


@pytest.mark.parametrize("bad, rc", [
    (dict(B=0), -1), (dict(T=0), -1), (dict(G=0), -1), (dict(H=0), -1), (dict(K=0), -1), (dict(V=-3), -1), (dict(H=3, G=2), -1),
    (dict(K=129), -4), (dict(V=200), -4), (dict(dtype=0), -4), (dict(dtype=7), -4), (dict(scale=float("nan")), -1),
    (dict(scale=float("inf")), -1), (dict(scale=1e39), -1), (dict(B=2**31), -4), (dict(T=2**31), -4), (dict(B=2**30, H=4), -4),
    (dict(q_stride=(0, -1, 0)), -1), (dict(k_stride=(-8, 8, 8)), -1), (dict(v_stride=(8, 8, -8)), -1),
    (dict(k_stride=(0, 1 << 24, 0)), -4), (dict(B=2**21), -4)])
def test_sizes_that_are_refused(lib, handle, bad, rc):
    d, n, one = _dims(**bad), C.c_size_t(), C.c_void_p(16)
    assert lib.kf_linear_attention_workspace(handle, C.byref(d), 0, C.byref(n)) == rc
    assert lib.kf_linear_attention(handle, C.byref(d), *[one] * 8, one, 1 << 30, None) == rc
    assert lib.kf_linear_attention_backward(handle, C.byref(d), *[one] * 13, one, 1 << 30, None) == rc
    if not {"T", "q_stride"} & set(bad) and bad.get("k_stride") != (0, 1 << 24, 0):
        assert lib.kf_linear_attention_step(handle, C.byref(d), *[one] * 5, 4, *[one] * 4, None) == rc
    assert lib.kf_last_error(handle)


def test_pointers_and_workspaces_that_are_refused(lib, handle):
    d, n, one = _dims(), C.c_size_t(), C.c_void_p(16)
    assert lib.kf_linear_attention(None, C.byref(d), *[one] * 8, one, 1 << 30, None) == -1
    assert lib.kf_linear_attention(handle, None, *[one] * 8, one, 1 << 30, None) == -1
    assert lib.kf_linear_attention_workspace(handle, C.byref(d), 0, None) == -1
    for i in (0, 1, 2, 3, 6):
        assert lib.kf_linear_attention(handle, C.byref(d), *[None if j == i else one for j in range(8)], one, 1 << 30, None) == -1
    for i in (0, 1, 2, 3, 6, 8, 9, 10, 11):
        assert lib.kf_linear_attention_backward(handle, C.byref(d), *[None if j == i else one for j in range(13)], one, 1 << 30, None) == -1
    assert lib.kf_linear_attention_workspace(handle, C.byref(d), 1, C.byref(n)) == 0 and n.value > 0
    assert lib.kf_linear_attention_backward(handle, C.byref(d), *[one] * 13, None, 0, None) == -3
    assert lib.kf_linear_attention_backward(handle, C.byref(d), *[one] * 13, one, n.value - 1, None) == -3
    assert lib.kf_linear_attention_backward(handle, C.byref(d), *[one] * 13, C.c_void_p(24), n.value, None) == -1
    d.g_o_stride[1] = -4
    assert lib.kf_linear_attention_backward(handle, C.byref(d), *[one] * 13, one, 1 << 30, None) == -1
    for i in (0, 1, 2, 3, 6, 7, 8):
        args = [None if j == i else one for j in range(10)]
        assert lib.kf_linear_attention_step(handle, C.byref(_dims()), *args[:5], 4, *args[6:], None) == -1
    for slots, count in ((one, 0), (one, -1), (one, 2**31), (None, 1)):
        assert lib.kf_linear_attention_step(handle, C.byref(_dims(B=2)), one, one, one, one, slots, count, *[one] * 4, None) == -1


def test_buffers_that_share_memory_are_refused(lib, handle):
    d, one, far = _dims(), C.c_void_p(1 << 12), C.c_void_p(1 << 30)
    state = 2 * 8 * 8 * 4  # bytes, of _dims()
    for off in (0, 4, state - 4, 4 - state):
        near = C.c_void_p((1 << 30) + off)
        assert lib.kf_linear_attention(handle, C.byref(d), one, one, one, one, far, None, one, near, one, 1 << 30, None) == -1
        assert b"overlaps" in lib.kf_last_error(handle)
        for s0, gs in ((far, None), (None, far)):
            assert lib.kf_linear_attention_backward(handle, C.byref(d), one, one, one, one, s0, None, one, gs, *[one] * 4, near, one, 1 << 30, None) == -1
            assert b"overlaps" in lib.kf_last_error(handle)
        if off:
            assert lib.kf_linear_attention_step(handle, C.byref(d), one, one, one, one, None, 1, far, near, one, one, None) == -1
            assert b"overlaps" in lib.kf_last_error(handle)
    coef = (C.c_double * 3)(1.5, -0.5, 0.0)
    for off in (0, 2, 5 * 96 * 96 * 2 - 2):
        assert lib.kf_orthogonalise(handle, 5, 96, 96, 2, 1, coef, 1e-7, far, C.c_void_p((1 << 30) + off), one, 1 << 40, None) == -1


@pytest.mark.parametrize("n, rows, cols, dtype, rc", [
    (0, 4, 4, 1, -1), (1, 0, 4, 1, -1), (1, 4, -1, 1, -1), (1, 4, 4, 4, -4), (1, 4, 4, -1, -4), (1, 1 << 18, 1 << 18, 1, -4),
    (1 << 40, 4, 4, 1, -4), (4, 1 << 17, 1 << 24, 1, -4), (1, 1 << 16, (1 << 15) + 1, 0, -4), (65536, 100, 100, 1, -4)])
def test_matrices_that_are_refused(lib, handle, n, rows, cols, dtype, rc):
    size, one = C.c_size_t(), C.c_void_p(16)
    coef = (C.c_double * 3)(1.5, -0.5, 0.0)
    assert lib.kf_orthogonalise_workspace(handle, n, rows, cols, dtype, C.byref(size)) == rc
    assert lib.kf_orthogonalise(handle, n, rows, cols, dtype, 1, coef, 1e-7, one, C.c_void_p(32), one, 1 << 40, None) == rc


def test_coefficients_that_are_refused(lib, handle):
    one, two = C.c_void_p(16), C.c_void_p(1 << 20)

    def call(coef, steps=None, eps=1e-7, M=one, X=two, ws=one):
        flat = np.asarray(coef, dtype=np.float64).ravel()
        return lib.kf_orthogonalise(handle, 1, 96, 96, 1, len(flat) // 3 if steps is None else steps,
                                    flat.ctypes.data_as(C.POINTER(C.c_double)), eps, M, X, ws, 0, None)

    assert call(NS5) == -3  # only the workspace is missing
    assert call([(1.5, -0.5, 0.0)] * 16) == -3
    assert call([(1.5, -0.5, 0.0)] * 17) == -1
    assert call(NS5, steps=0) == -1
    assert call(NS5, eps=-1.0) == -1 and call(NS5, eps=float("nan")) == -1 and call(NS5, eps=float("inf")) == -1
    assert call(NS5, M=None) == -1 and call(NS5, X=None) == -1 and call(NS5, X=one) == -1
    assert call([(float("nan"), 0, 0)]) == -1 and call([(1.0, 0, 2e3)]) == -1
    assert call([(2.0, 0, 0)]) == -1            # carries the value 1 to 2
    assert call([(1.2, 0, 0)] * 3) == -3        # 1.728
    assert call([(1.2, 0, 0)] * 4) == -1        # 2.07
    assert call([(4.0, -4.0, 0.0)]) == -3       # top inside the interval: 1.54 at s = 0.577
    assert call([(6.0, -6.0, 0.0)]) == -1       # 2.31 there, 0 at both ends


@pytest.mark.parametrize("coef", [(6.0, -6.0, 1e-17), (100.0, -100.0, 1e-16), (100.0, -100.0, -1e-16), (6.0, -6.0, 1e-300), (-6.0, 6.0, 1e-17)])
def test_a_quintic_that_is_nearly_a_cubic_is_refused(lib, handle, coef):
    """The maximum inside the interval is found however small the quintic's own coefficient: 2.31 and 38 at s = 0.577."""
    one, two = C.c_void_p(16), C.c_void_p(1 << 20)
    assert lib.kf_orthogonalise(handle, 1, 96, 96, 1, 1, (C.c_double * 3)(*coef), 1e-7, one, two, one, 1 << 40, None) == -1
    assert b"singular value" in lib.kf_last_error(handle)


# a published list of steps, each the best on what the one before leaves; the first reaches 1.992
OPTIMISED = [(8.28721201814563, -23.595886519098837, 17.300387312530933), (4.107059111542203, -2.9478499167379106, 0.5448431082926601),
             (3.9486908534822946, -2.908902115962949, 0.5518191394370137), (3.3184196573706015, -2.488488024314874, 0.51004894012372),
             (2.300652019954817, -1.6689039845747493, 0.4188073119525673), (1.891301407787398, -1.2679958271945868, 0.37680408948524835),
             (1.875, -1.25, 0.375)]


@pytest.mark.parametrize("safety", [1.0, 1.01])
@pytest.mark.parametrize("rows, cols, dtype", [(96, 96, 1), (96, 96, 2), (96, 96, 0), (300, 200, 3)])
def test_steps_that_come_close_to_two_are_taken(lib, handle, rows, cols, dtype, safety):
    coef = [x for a, b, c in OPTIMISED for x in (a / safety, b / safety ** 3, c / safety ** 5)]
    one, two = C.c_void_p(16), C.c_void_p(1 << 20)
    assert lib.kf_orthogonalise(handle, 1, rows, cols, dtype, len(OPTIMISED), (C.c_double * len(coef))(*coef), 1e-7, one, two, None, 0, None) == -3


def test_the_bound_of_a_step_is_its_polynomials_maximum(lib, handle):
    """Random lists: refused exactly where a fine grid finds a value above the bound in some step.  (The workspace is left out, so that
    a list that is taken ends there.)"""
    rng = np.random.default_rng(6)
    one, two = C.c_void_p(16), C.c_void_p(1 << 20)
    taken = 0
    for _ in range(2000):
        coef = rng.uniform(-6, 6, 3) * np.where(rng.random(3) < 0.5, 1.0, 10.0 ** -rng.integers(0, 18, 3))
        s = np.linspace(0.0, 1.0, 4001)
        top = np.abs(s * (coef[0] + s * s * (coef[1] + s * s * coef[2]))).max()
        if 1.85 < top < 2.05:  # (on the bound, or a grid's step away from it)
            continue
        rc = lib.kf_orthogonalise(handle, 1, 96, 96, 1, 1, (C.c_double * 3)(*coef), 1e-7, one, two, None, 0, None)
        assert rc == (-3 if top < 1.9 else -1), (coef, top)
        taken += rc == -3
    assert 200 < taken < 1900


# ---------------------------------------------------------------------------------------------- refusals, in the engine
@pytest.fixture
def engine():
    from pymc_statespace_amd import KalmanEngine

    eng = object.__new__(KalmanEngine)  # (a real one needs a GPU; the checks below come before any call)
    eng.device = torch.device("cpu")
    eng._h = None
    return eng


def test_shapes_and_types_that_the_engine_refuses(engine):
    q, v, g = torch.zeros(2, 5, 1, 8), torch.zeros(2, 5, 2, 8), torch.zeros(2, 5, 2)
    go = torch.zeros(2, 5, 2, 8)
    for bad in ((q[0], q, v, g), (q, q[:, :4], v, g), (q, q, v[:1], g), (q, q, v, g[:, :4]), (q, q, v, torch.zeros(3))):
        with pytest.raises(ValueError):
            engine.linear_attention(*bad)
        with pytest.raises(ValueError):
            engine.linear_attention_backward(*bad, go)
    for bad in ((q.double(), q, v, g), (q, q.bfloat16(), v, g), (q, q, v.half(), g), (q.to(torch.int32),) * 2 + (v, g)):
        with pytest.raises(TypeError):
            engine.linear_attention(*bad)
    with pytest.raises(ValueError):
        engine.linear_attention(q, q, v, g, initial_state=torch.zeros(2, 2, 8, 7))
    with pytest.raises(ValueError):
        engine.linear_attention(q, q, v, g, lengths=torch.zeros(2))
    with pytest.raises(ValueError):
        engine.linear_attention(q, q, v, g, lengths=torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError):
        engine.linear_attention_backward(q, q, v, g, go[..., :7])
    with pytest.raises(TypeError):
        engine.linear_attention_backward(q, q, v, g, go.bfloat16())


def test_states_that_the_engine_refuses(engine):
    q, v, g = torch.zeros(2, 1, 8), torch.zeros(2, 2, 8), torch.zeros(2, 2)
    for state in (torch.zeros(2, 2, 8, 8).double(), torch.zeros(2, 2, 8, 7), torch.zeros(2, 2, 8, 16)[..., ::2], np.zeros((2, 2, 8, 8), np.float32)):
        with pytest.raises(ValueError):
            engine.linear_attention_step(q, q, v, g, state)
    pool = torch.zeros(5, 2, 8, 8)
    with pytest.raises(ValueError):
        engine.linear_attention_step(q, q, v, g, pool[:4], state_out=pool[1:])
    with pytest.raises(ValueError):
        engine.linear_attention_step(q, q, v, g, pool, state_out=pool[:4].clone())
    with pytest.raises(ValueError):
        engine.linear_attention_step(q, q, v, g, pool, slots=torch.zeros(3, dtype=torch.int32))


def test_matrices_that_the_engine_refuses(engine):
    with pytest.raises(TypeError):
        engine.orthogonalise(torch.zeros(3, 3, dtype=torch.int32))
    with pytest.raises(ValueError):
        engine.orthogonalise(torch.zeros(3))
    with pytest.raises(ValueError):
        engine.orthogonalise(torch.zeros(0, 3, 3))
    with pytest.raises(ValueError):
        engine.orthogonalise(torch.zeros(3, 3), steps=0)
    with pytest.raises(ValueError):
        engine.orthogonalise(torch.zeros(3, 3), steps=17)
    with pytest.raises(ValueError):
        engine.orthogonalise(torch.zeros(3, 3), coefficients=[(1.0, 2.0)])


@pytest.mark.parametrize("steps", [2.5, "3", None, float("nan")])
@pytest.mark.parametrize("coefficients", [(1.5, -0.5, 0.0), [1.5, -0.5, 0.0]])
def test_a_number_of_steps_that_is_not_whole_is_refused(engine, steps, coefficients):
    with pytest.raises((TypeError, ValueError)):
        engine.orthogonalise(torch.zeros(3, 3), steps=steps, coefficients=coefficients)


def test_steps_as_any_whole_number():
    from pymc_statespace_amd.engine import _newton_schulz

    want = [1.5, -0.5, 0.25] * 3
    for steps in (3, 3.0, np.int64(3), torch.tensor(3)):
        for c in ((1.5, -0.5, 0.25), [1.5, -0.5, 0.25], np.array([1.5, -0.5, 0.25])):
            n, coef = _newton_schulz(c, steps)
            assert n == 3 and list(coef) == want
