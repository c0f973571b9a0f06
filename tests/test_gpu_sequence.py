"""Sequence operators on the GPU against their definitions in 64 bits (oracle/sequence_numpy.py).

Tolerances.  An output in a 16-bit type is rounded once at its end (half a step: u = finfo.eps / 2), and a 16-bit factor inside
(the masked scores, the state as an operand) once more, each relative to the terms of the sum it enters: at most
u |out| + 2 u A with A the same sum over absolute values.  Sums in 32 bits over n terms are off by at most n 2^-24 A, with n = the
longest chain: K or V terms of a product, 64 tokens of a chunk, and three roundings for each chunk that a state passes through.
A is the oracle's own recurrence on the absolute values."""
import numpy as np
import pytest
import torch

from oracle import sequence_numpy as sn

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
NS = (3.4445, -4.7750, 2.0315)


@pytest.fixture(scope="module")
def eng():
    from pymc_statespace_amd import get_engine

    return get_engine()


def _u(dtype):
    return torch.finfo(dtype).eps / 2


def _least(dtype):
    """Below a type's smallest normal number its steps no longer shrink: half of one, whatever the value (fp16: 2^-25, met below
    2^-14; never met in the other types here)."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def _terms(T, K, V):
    return K + V + 64 + 3 * (T // 32 + 2) + 32


def _make(seed, B, T, G, H, K, V, dtype, per_token=True, init=True, reset=0.0):
    """float64 numpy arrays whose values `dtype` holds exactly."""
    rng = np.random.default_rng(seed)

    def r(*shape):
        return torch.from_numpy(rng.standard_normal(shape)).to(dtype).double().numpy()

    p = dict(q=r(B, T, G, K), k=r(B, T, G, K), v=r(B, T, H, V), g_o=r(B, T, H, V), scale=0.5 / np.sqrt(K))
    base = -np.exp(rng.uniform(np.log(1e-3), np.log(2.0), H))
    g = base * np.exp(0.5 * rng.standard_normal((B, T, H))) if per_token else base
    p["log_decay"] = g.astype(np.float32).astype(np.float64)
    if reset:
        p["log_decay"][rng.random(p["log_decay"].shape) < reset] = -np.inf
    p["s0"] = rng.standard_normal((B, H, K, V)).astype(np.float32).astype(np.float64) if init else None
    p["g_sT"] = rng.standard_normal((B, H, K, V)).astype(np.float32).astype(np.float64) if init else None
    return p


def _dev(x, dtype=torch.float32):
    return None if x is None else torch.from_numpy(np.asarray(x)).to("cuda", dtype)


def _forward(eng, p, dtype, lengths=None):
    return eng.linear_attention(_dev(p["q"], dtype), _dev(p["k"], dtype), _dev(p["v"], dtype), _dev(p["log_decay"]), scale=p["scale"],
                                initial_state=_dev(p["s0"]), lengths=lengths)


def _backward(eng, p, dtype, lengths=None):
    return eng.linear_attention_backward(_dev(p["q"], dtype), _dev(p["k"], dtype), _dev(p["v"], dtype), _dev(p["log_decay"]),
                                         _dev(p["g_o"], dtype), scale=p["scale"], initial_state=_dev(p["s0"]), lengths=lengths,
                                         g_final_state=_dev(p["g_sT"]))


def _abs(x):
    return None if x is None else np.abs(x)


def _near(got, want, tol, what):
    got = got.double().cpu().numpy()
    assert got.shape == want.shape, what
    assert np.isfinite(got).all(), what
    worst = np.max(np.abs(got - want) - tol)
    assert worst <= 0, f"{what}: {np.max(np.abs(got - want)):.3e} off, {worst:.3e} beyond the bound"


def _check_forward(eng, p, dtype, lengths=None):
    B, T, H, V = p["v"].shape
    K = p["q"].shape[-1]
    host = None if lengths is None else np.asarray(lengths)
    dev = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    o, S = _forward(eng, p, dtype, dev)
    ro, rS = sn.attention(p["q"], p["k"], p["v"], p["log_decay"], p["scale"], p["s0"], host)
    ao, aS = sn.attention(_abs(p["q"]), _abs(p["k"]), _abs(p["v"]), p["log_decay"], p["scale"], _abs(p["s0"]), host)
    u, n = _u(dtype), _terms(T, K, V) * U32
    inner = 0 if dtype == torch.float32 else 2 * u
    _near(o, ro, u * np.abs(ro) + (inner + n) * ao + _least(dtype), "o")
    _near(S, rS, n * aS + 1e-30, "state")
    return o, S


def _check_backward(eng, p, dtype, lengths=None):
    B, T, H, V = p["v"].shape
    G, K = p["q"].shape[2:]
    host = None if lengths is None else np.asarray(lengths)
    dev = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    got = _backward(eng, p, dtype, dev)
    args = ("q", "k", "v", "log_decay", "g_o")
    ref = sn.attention_gradient(*(p[x] for x in args), p["scale"], p["s0"], host, p["g_sT"])
    mag = sn.attention_gradient(*(p[x] if x == "log_decay" else _abs(p[x]) for x in args), p["scale"], _abs(p["s0"]), host, _abs(p["g_sT"]))
    u, n = _u(dtype), (_terms(T, K, V) + H // G) * U32
    inner = 0 if dtype == torch.float32 else 2 * u
    for x in ("q", "k", "v"):
        _near(got[x], ref[x], u * np.abs(ref[x]) + (inner + n) * mag[x] + _least(dtype), "d" + x)
    if p["s0"] is not None:
        _near(got["initial_state"], ref["initial_state"], n * mag["initial_state"] + 1e-30, "dS0")
    else:
        assert got["initial_state"] is None
    # d log a: pairs inside a chunk are summed as a running difference, of the size of what the chunk's tokens read and write.  (In
    # the products with the states 16-bit types take them in exact parts: nothing is added to the sums' own roundings.)
    per = H // G
    aq, ak = np.repeat(_abs(p["q"]), per, 2), np.repeat(_abs(p["k"]), per, 2)
    single = sn.attention_gradient(aq, ak, _abs(p["v"]), np.broadcast_to(p["log_decay"], (B, T, H)), _abs(p["g_o"]), p["scale"],
                                   _abs(p["s0"]), host, _abs(p["g_sT"]))
    size = (aq * single["q"]).sum(-1) + (ak * single["k"]).sum(-1)
    size = np.concatenate([size, np.zeros((B, 64, H))], 1)
    size = np.stack([size[:, t:t + 64].sum(1) for t in range(T)], 1) + single["log_decay"]
    bound = n * size
    if p["log_decay"].ndim == 1:
        bound = bound.sum((0, 1))
    _near(got["log_decay"], ref["log_decay"], bound + 1e-30, "d log_decay")
    return got


SHAPES = [  # B, T, G, H, K, V
    (1, 1, 1, 1, 1, 1), (2, 3, 1, 2, 5, 7), (1, 64, 2, 2, 16, 16), (2, 65, 1, 3, 33, 40), (1, 130, 2, 4, 64, 64), (2, 200, 1, 1, 128, 128),
    (1, 257, 3, 3, 100, 20), (3, 127, 2, 2, 8, 128), (1, 31, 1, 1, 128, 65), (1, 129, 1, 8, 24, 96)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward(eng, shape, dtype):
    _check_forward(eng, _make(1, *shape, TYPES[dtype]), TYPES[dtype])


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_backward(eng, shape, dtype):
    _check_backward(eng, _make(2, *shape, TYPES[dtype]), TYPES[dtype])


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("per_token, init, lengths", [(False, False, None), (True, False, [70, 0, 1]), (False, True, [130, 64, 63]),
                                                      (True, True, [0, 0, 0]), (True, True, [999, -5, 65])])
def test_fixed_decays_no_state_and_padded_batches(eng, dtype, per_token, init, lengths):
    p = _make(3, 3, 130, 2, 4, 40, 72, TYPES[dtype], per_token=per_token, init=init)
    _check_forward(eng, p, TYPES[dtype], lengths)
    _check_backward(eng, p, TYPES[dtype], lengths)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_resets(eng, dtype):
    """A log decay of -infinity empties the state: nothing of what came before is left, and no inf - inf."""
    p = _make(4, 2, 150, 1, 2, 32, 48, TYPES[dtype], reset=0.1)
    _check_forward(eng, p, TYPES[dtype])
    _check_backward(eng, p, TYPES[dtype])
    p["log_decay"][:] = -np.inf
    _check_forward(eng, p, TYPES[dtype])
    _check_backward(eng, p, TYPES[dtype])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_long_sequence(eng, dtype):
    """Long enough that the time axis is split over workgroups."""
    p = _make(5, 1, 3001, 1, 2, 24, 40, TYPES[dtype])
    _check_forward(eng, p, TYPES[dtype])
    _check_backward(eng, p, TYPES[dtype])


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", [(1, 1100, 2, 2, 5, 70), (1, 1100, 1, 3, 77, 3)], ids=str)
def test_long_and_narrow(eng, shape, dtype):
    """Rows shorter than 16 bytes, over many segments."""
    p = _make(15, *shape, TYPES[dtype])
    _check_forward(eng, p, TYPES[dtype])
    _check_backward(eng, p, TYPES[dtype])


@pytest.mark.parametrize("dtype", list(TYPES))
def test_decays_that_grow(eng, dtype):
    """Positive log decays are a growth, as the recurrence has it."""
    p = _make(16, 2, 200, 1, 2, 24, 40, TYPES[dtype])
    p["log_decay"] = np.random.default_rng(17).uniform(-0.05, 0.04, p["log_decay"].shape).astype(np.float32).astype(np.float64)
    _check_forward(eng, p, TYPES[dtype])
    _check_backward(eng, p, TYPES[dtype])


# many heads: (B, T, G, H, K, V), fixed decays, lengths, and (segments, chunks of each) of the gradient by data type on 256 units
MANY = [((2, 300, 16, 64, 72, 72), True, [300, 131], (2, 3), (2, 5)),       # 128 x 128, segments summed by the workgroups that need them
        ((4, 200, 64, 64, 100, 128), True, None, (1, 4), (1, 7)),           # one segment
        ((2, 1100, 8, 32, 64, 40), True, [1100, 577], (6, 3), (7, 5)),      # 64 x 64
        ((2, 2500, 16, 16, 32, 24), False, None, (20, 2), (27, 3)),         # 32 x 32, more than 8 segments: summed by a launch of their own
        ((3, 2100, 3, 12, 20, 32), True, [2100, 0, 1027], (17, 2), (22, 3)),  # the same, ragged
        ((4, 260, 16, 32, 4, 7), False, [260, 64, 65, 1], (2, 3), (2, 5))]  # rows shorter than 16 bytes


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape, per_token, lengths, split16, split32", MANY, ids=lambda x: str(x) if isinstance(x, tuple) and len(x) == 6 else "")
def test_several_chunks_in_each_segment(eng, monkeypatch, shape, per_token, lengths, split16, split32, dtype):
    """Batches of so many heads that a workgroup of the gradient walks several chunks: states kept at every chunk's start, both sums
    carried from chunk to chunk."""
    import ctypes as C

    from oracle import sequence_torch as st
    from pymc_statespace_amd import _lib

    B, T, G, H, K, V = shape
    t = TYPES[dtype]
    # the split that the case is for, from what the call asks for: a state for each chunk's start is kept where segments have several
    chunk = 64 if dtype == "bf16" else 32
    D = 128 if min(K, V) < 8 else next(d for d in (32, 64, 128) if max(K, V) <= d)
    segments, each = split16 if dtype == "bf16" else split32
    if torch.cuda.get_device_properties(0).multi_processor_count == 256:
        chunks, up = -(-T // chunk), lambda n: -(-n // 256) * 256
        assert each > 1 and (segments - 1) * each < chunks <= segments * each
        want = 2 * up(B * H * (segments - 1) * D * D * 4) + up(B * H * segments * 4) + 2 * up(B * H * (segments - 1) * 4) + up(B * H * chunks * D * D * 4) \
            + (2 * up(B * T * H * K * 4) if G != H else 0) + (0 if per_token else up(B * H * segments * 8))
        dims, n = _lib.pack_attention_dims(B, T, G, H, K, V, _lib.KF_DTYPE[{"f32": "float32", "f16": "float16", "bf16": "bfloat16"}[dtype]], per_token,
                                           1.0, *[0] * 12), C.c_size_t()
        assert eng.lib.kf_linear_attention_workspace(eng._h, dims, 1, C.byref(n)) == 0 and n.value == want
    # (the oracle's own loops over tokens and sequences would take minutes)
    for name in ("attention", "attention_gradient"):
        monkeypatch.setattr(sn, name, lambda *a, f=getattr(st, name): f(*a, device="cuda"))
    p = _make(19, *shape, t, per_token=per_token)
    _check_forward(eng, p, t, lengths)
    _check_backward(eng, p, t, lengths)
    if lengths is not None:  # the same bits without what lies behind the sequences
        dev = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        want = _backward(eng, p, t, dev)
        for b, n in enumerate(lengths):
            for name in ("q", "k", "v", "g_o") + (("log_decay",) if per_token else ()):
                p[name][b, n:] = np.nan
        got = _backward(eng, p, t, dev)
        assert all(torch.equal(want[n], got[n]) for n in want)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("H", [2, 64])
def test_a_growth_that_nothing_takes_part_in(eng, monkeypatch, H, dtype):
    """Decays of e^0.5 a token over 1500 tokens: far more than fp32 holds over a segment or all of them, but the state is zero until token
    700 and after the reset at 800, and so is what flows back from behind it and to before the reset at 690.  (H: segments summed by a
    launch of their own, and by the workgroups that need them.)"""
    from oracle import sequence_torch as st

    for name in ("attention", "attention_gradient"):
        monkeypatch.setattr(sn, name, lambda *a, f=getattr(st, name): f(*a, device="cuda"))
    p = _make(26, 1, 1500, H, H, 24, 40, TYPES[dtype], init=False)
    p["log_decay"] = np.random.default_rng(27).uniform(0.48, 0.52, p["log_decay"].shape).astype(np.float32).astype(np.float64)
    p["log_decay"][:, [690, 800]] = -np.inf
    p["k"][:, :700] = p["k"][:, 780:] = 0.0
    p["g_o"][:, :700] = p["g_o"][:, 800:] = 0.0
    if dtype == "f16":  # (e^50 does not fit its outputs: the state and its gradient, which are fp32, by values that keep them small)
        for x in ("k", "g_o"):
            p[x] = torch.from_numpy(p[x] * 2.0 ** -14).half().double().numpy()
        p["log_decay"][:, 700:800] *= 0.25
        p["log_decay"] = p["log_decay"].astype(np.float32).astype(np.float64)
    _check_forward(eng, p, TYPES[dtype])
    _check_backward(eng, p, TYPES[dtype])


def test_no_decay_at_all(eng):
    """log_decay = 0: a plain running sum, the state grows with the length."""
    p = _make(6, 1, 700, 1, 1, 16, 16, torch.float32)
    p["log_decay"][:] = 0.0
    _check_forward(eng, p, torch.float32)
    _check_backward(eng, p, torch.float32)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_what_lies_behind_a_sequence_is_not_read(eng, dtype):
    p = _make(7, 2, 100, 1, 2, 20, 24, TYPES[dtype])
    lengths = torch.tensor([37, 100], dtype=torch.int32, device="cuda")
    want, wg = _forward(eng, p, TYPES[dtype], lengths), _backward(eng, p, TYPES[dtype], lengths)
    for name in ("q", "k", "v", "g_o", "log_decay"):
        p[name][0, 37:] = np.nan
    got, gg = _forward(eng, p, TYPES[dtype], lengths), _backward(eng, p, TYPES[dtype], lengths)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    for name in wg:
        assert torch.equal(wg[name], gg[name]), name
    assert not got[0][0, 37:].any() and not gg["v"][0, 37:].any() and not gg["log_decay"][0, 37:].any()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("name", ["q", "k", "v", "log_decay"])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
def test_a_later_token_never_reaches_an_earlier_one(eng, dtype, name, value):
    """NaN and infinities in a token's values stay out of all rows before it, also of its own chunk."""
    if name == "log_decay" and not np.isnan(value):
        pytest.skip("a decay of -inf is a reset, one of +inf is outside the range")
    p = _make(8, 1, 150, 1, 2, 24, 40, TYPES[dtype])
    want, _ = _forward(eng, p, TYPES[dtype])
    at = 83
    p[name][0, at] = value
    got, _ = _forward(eng, p, TYPES[dtype])
    assert torch.equal(got[:, :at], want[:, :at])
    assert not torch.isfinite(got[:, at]).all()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("sign", [1, -1])
def test_values_up_to_the_types_largest_next_to_a_nan(eng, dtype, sign):
    """A value of the type's largest size is finite: beside a token that is not, it counts once, as without that token."""
    t, at = TYPES[dtype], 83
    p = _make(18, 1, 150, 1, 2, 24, 40, t)
    # weights exp(..) s (q . k) below 1 / 8, and a state that stays finite: |k| <= 1e-3
    p["k"] = torch.from_numpy(1e-3 * np.clip(p["k"], -1, 1)).to(t).double().numpy()
    p["q"] = torch.from_numpy(np.clip(p["q"], -1, 1)).to(t).double().numpy()
    p["s0"] = None
    p["v"][0, 70, :, ::3] = sign * torch.finfo(t).max
    want, _ = _forward(eng, p, t)
    assert torch.isfinite(want).all() and float(want[0, 70:].abs().max()) > 1.0
    p["v"][0, at] = np.nan
    got, _ = _forward(eng, p, t)
    assert torch.equal(got[:, :at], want[:, :at])
    assert torch.isnan(got[:, at:]).all()
    # and in rows that see both: the NaN reaches one head's columns only where it stands
    p["v"][0, at] = 0.0
    clean, _ = _forward(eng, p, t)
    p["v"][0, at, 0, 1] = np.inf
    got, _ = _forward(eng, p, t)
    keep = np.arange(40) != 1
    # columns without the infinity: the same sums, their terms in another order (the products, and what is added to them)
    off = (got[:, :, 0][..., keep].double() - clean[:, :, 0][..., keep].double()).abs()
    u = _u(t)
    ao, _ = sn.attention(_abs(p["q"]), _abs(p["k"]), np.where(np.isfinite(p["v"]), np.abs(p["v"]), 0.0), p["log_decay"], p["scale"])
    bound = torch.from_numpy(2 * (u + (0 if t == torch.float32 else 2 * u) + _terms(150, 24, 40) * U32) * ao[:, :, 0][..., keep]).cuda() + 2 * _least(t)
    assert (off <= bound).all()
    assert torch.equal(got[:, :, 1], clean[:, :, 1])


@pytest.mark.parametrize("dtype", list(TYPES))
def test_views_of_a_fused_projection(eng, dtype):
    """q, k, v as slices of one tensor, heads before tokens, odd offsets: strides are read, nothing is assumed of alignment."""
    t, p = TYPES[dtype], _make(9, 2, 77, 2, 4, 24, 40, TYPES[dtype])
    fused = torch.zeros(2, 77, 1 + 2 * 2 * 24 + 4 * 40, device="cuda", dtype=t)
    q, k, v = (_dev(p[x], t) for x in ("q", "k", "v"))
    fq, fk = fused[..., 1:49].unflatten(-1, (2, 24)), fused[..., 49:97].unflatten(-1, (2, 24))
    fv, go = fused[..., 97:].unflatten(-1, (4, 40)), _dev(p["g_o"], t)
    fq.copy_(q), fk.copy_(k), fv.copy_(v)
    g = _dev(p["log_decay"])
    want, ws = eng.linear_attention(q, k, v, g)
    wg = eng.linear_attention_backward(q, k, v, g, go)
    other = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v, go)]
    last = [x.transpose(-1, -2).contiguous().transpose(-1, -2) for x in (q, k, v, go)]
    for a, b, c, d in ((fq, fk, fv, go), tuple(other), tuple(last)):
        o, s = eng.linear_attention(a, b, c, g)
        assert torch.equal(o, want) and torch.equal(s, ws)
        grads = eng.linear_attention_backward(a, b, c, g, d)
        for n in ("q", "k", "v", "log_decay"):
            assert torch.equal(grads[n], wg[n]), n
    # one query row for every token and group (stride 0)
    e = q[:, :1, :1].expand(2, 77, 2, 24)
    a, b = eng.linear_attention(e, k, v, g), eng.linear_attention(e.contiguous(), k, v, g)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_gradient_against_differences(eng, dtype):
    """Along random directions in fp32 inputs: the change of the loss, computed by the forward kernel itself."""
    if dtype == "bf16":
        pytest.skip("a difference needs more digits than bf16 outputs have; the gradient is checked against the formula")
    p = _make(10, 1, 90, 1, 2, 16, 24, torch.float32)
    grad = _backward(eng, p, torch.float32)
    rng = np.random.default_rng(3)

    def loss(x):
        o, S = _forward(eng, x, torch.float32)
        return float((o.double().cpu().numpy() * p["g_o"]).sum() + (S.double().cpu().numpy() * p["g_sT"]).sum())

    sizes = sn.attention(_abs(p["q"]), _abs(p["k"]), _abs(p["v"]), p["log_decay"], p["scale"], _abs(p["s0"]))
    noise = _terms(90, 16, 24) * U32 * ((sizes[0] * _abs(p["g_o"])).sum() + (sizes[1] * _abs(p["g_sT"])).sum())
    for name, key in (("q", "q"), ("k", "k"), ("v", "v"), ("log_decay", "log_decay"), ("s0", "initial_state")):
        step = 1e-2 * rng.standard_normal(p[name].shape)
        hi, lo = (p | {name: (p[name] + s * step).astype(np.float32).astype(np.float64)} for s in (1, -1))
        want = loss(hi) - loss(lo)
        have = float((grad[key].double().cpu().numpy() * (hi[name] - lo[name])).sum())
        # linear in q, v, s0 and k; cubic terms of the decays: |step|^3 / 3 of the size of the gradient's terms
        cubic = 0.0 if name != "log_decay" else 1e-4 * float((grad[key].abs().double().cpu().numpy() * np.abs(step)).sum()) * 50
        assert abs(want - have) <= 2 * noise + cubic, (name, want, have)


def test_the_same_bits_every_time(eng):
    for dtype in TYPES.values():
        p = _make(11, 2, 300, 2, 4, 64, 64, dtype)
        a, b = _forward(eng, p, dtype), _forward(eng, p, dtype)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        ga, gb = _backward(eng, p, dtype), _backward(eng, p, dtype)
        assert all(torch.equal(ga[n], gb[n]) for n in ga)


# ------------------------------------------------------------------------------------------------------ single tokens
def _step_problem(seed, B, N, G, H, K, V, dtype, per_row=True):
    p = _make(seed, B, 1, G, H, K, V, dtype, per_token=per_row)
    rng = np.random.default_rng(seed + 1)
    return dict(q=p["q"][:, 0], k=p["k"][:, 0], v=p["v"][:, 0], g=p["log_decay"][:, 0] if per_row else p["log_decay"], scale=p["scale"],
                state=rng.standard_normal((N, H, K, V)).astype(np.float32).astype(np.float64))


def _check_step(eng, p, dtype, slots=None, in_place=False):
    K, V = p["q"].shape[-1], p["v"].shape[-1]
    state = _dev(p["state"])
    out = None if in_place else torch.full_like(state, 7.0)
    dev = None if slots is None else torch.tensor(slots, dtype=torch.int32, device="cuda")
    o, info = eng.linear_attention_step(_dev(p["q"], dtype), _dev(p["k"], dtype), _dev(p["v"], dtype), _dev(p["g"]), state,
                                        scale=p["scale"], slots=dev, state_out=out)
    ro, rS = sn.attention_step(p["q"], p["k"], p["v"], p["g"], p["state"], p["scale"], slots)
    ao, aS = sn.attention_step(_abs(p["q"]), _abs(p["k"]), _abs(p["v"]), p["g"], _abs(p["state"]), p["scale"], slots)
    n = _terms(len(p["v"]), K, V) * U32
    _near(o, ro, _u(dtype) * np.abs(ro) + n * ao + _least(dtype), "o")
    got = state if in_place else out
    used = range(len(p["v"])) if slots is None else [s for s in set(slots) if 0 <= s < len(p["state"])]
    rest = [s for s in range(len(p["state"])) if s not in set(used)]
    if used:
        _near(got[list(used)], rS[list(used)], n * aS[list(used)] + 1e-30, "state")
    assert torch.equal(got[rest], _dev(p["state"])[rest] if in_place else torch.full_like(got[rest], 7.0))
    if not in_place:
        assert torch.equal(state, _dev(p["state"]))
    want = [0] * len(p["v"]) if slots is None else [int(s >= len(p["state"])) for s in slots]
    assert info.tolist() == want
    return o


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 1, 1), (3, 3, 1, 2, 5, 7), (2, 2, 2, 4, 64, 64), (5, 5, 1, 1, 128, 128), (2, 2, 2, 2, 100, 33),
                                   (1, 1, 4, 8, 48, 100), (70, 70, 1, 1, 4, 12)], ids=str)
@pytest.mark.parametrize("in_place", [False, True])
def test_step(eng, shape, dtype, in_place):
    _check_step(eng, _step_problem(20, *shape, TYPES[dtype]), TYPES[dtype], in_place=in_place)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("slots", [[4, 0, 2], [-1, -1, -1], [5, -1, 1], [9, 10, 2**31 - 1], [3, 3, 3], [1, 5, 1], [0, -1, 0]], ids=str)
def test_step_in_a_pool(eng, dtype, slots):
    for per_row in (True, False):
        _check_step(eng, _step_problem(21, 3, 9, 2, 4, 24, 40, TYPES[dtype], per_row), TYPES[dtype], slots=slots)
        _check_step(eng, _step_problem(22, 3, 9, 2, 4, 64, 64, TYPES[dtype], per_row), TYPES[dtype], slots=slots, in_place=True)


def test_step_many_rows_of_one_slot(eng):
    rng = np.random.default_rng(5)
    slots = rng.integers(-1, 4, 300).tolist()
    _check_step(eng, _step_problem(23, 300, 4, 1, 2, 16, 20, torch.float32), torch.float32, slots=slots)


def test_step_far_into_a_pool(eng):
    """An offset over 2^31 elements: the last of 140000 slots of 16384 values."""
    K = V = 64
    state = torch.zeros(140000, 4, K, V, device="cuda")
    p = _step_problem(24, 2, 2, 1, 4, K, V, torch.bfloat16)
    slots = torch.tensor([139999, 0], dtype=torch.int32, device="cuda")
    state[139999], state[0] = _dev(p["state"][0]), _dev(p["state"][1])
    small = _dev(p["state"])
    args = [_dev(p[x], torch.bfloat16) for x in ("q", "k", "v")] + [_dev(p["g"])]
    o, _ = eng.linear_attention_step(*args, state, slots=slots)
    want, _ = eng.linear_attention_step(*args, small)
    assert torch.equal(o, want) and torch.equal(state[139999], small[0]) and torch.equal(state[0], small[1])
    assert not state[1:139999].any()


@pytest.mark.parametrize("dtype", list(TYPES))
def test_a_prompt_then_single_tokens(eng, dtype):
    """The forms agree with each other and with the whole sequence: a prompt in two pieces, then tokens one at a time."""
    t, p = TYPES[dtype], _make(12, 2, 200, 1, 2, 40, 56, TYPES[dtype], init=False)
    q, k, v, g = _dev(p["q"], t), _dev(p["k"], t), _dev(p["v"], t), _dev(p["log_decay"])
    ro, rS = sn.attention(p["q"], p["k"], p["v"], p["log_decay"], p["scale"])
    ao, aS = sn.attention(_abs(p["q"]), _abs(p["k"]), _abs(p["v"]), p["log_decay"], p["scale"])
    parts, state = [], None
    for lo, hi in ((0, 91), (91, 190)):
        o, state = eng.linear_attention(q[:, lo:hi], k[:, lo:hi], v[:, lo:hi], g[:, lo:hi], scale=p["scale"], initial_state=state)
        parts.append(o)
    for i in range(190, 200):
        o, _ = eng.linear_attention_step(q[:, i], k[:, i], v[:, i], g[:, i], state, scale=p["scale"])
        parts.append(o[:, None])
    u, n = _u(t), (_terms(200, 40, 56) + 30) * U32
    _near(torch.cat(parts, 1), ro, u * np.abs(ro) + ((0 if t == torch.float32 else 2 * u) + n) * ao + _least(t), "o")
    _near(state, rS, n * aS, "state")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_as_many_sequences_as_are_allowed(eng, dtype):
    """B H = 2^22 - 1 with as many tiles of V as there can be; one token each: S = k v', o = s q k v."""
    B, V = 2 ** 22 - 1, 100
    gen = torch.Generator(device="cuda").manual_seed(25)
    q, k = (torch.randn(B, 1, 1, 1, device="cuda", generator=gen).to(dtype) for _ in range(2))
    v = torch.randn(B, 1, 1, V, device="cuda", generator=gen).to(dtype)
    o, state = eng.linear_attention(q, k, v, torch.zeros(1, device="cuda"), scale=0.5)
    # one rounded product each (the state), and for o the score, rounded as the type is, times v, rounded to it
    want = k.float() * v.float()
    assert bool(((state[:, :, 0] - want[:, 0]).abs() <= 2 * U32 * want[:, 0].abs()).all())
    want = 0.5 * q.double() * k.double() * v.double()
    assert bool(((o.double() - want).abs() <= (2 * _u(dtype) + 4 * U32) * want.abs() * (1 + _u(dtype)) + 1e-37).all())
    with pytest.raises(Exception, match="B H"):
        x = torch.zeros(1, device="cuda", dtype=dtype).expand(2 ** 22, 1, 1, 1)
        eng.linear_attention(x, x, x, torch.zeros(1, device="cuda"))


# ------------------------------------------------------------------------------------------------ orthogonalised updates
def _amplified(S, coefficients):
    """How far an error of relative size 1 (of |X|_F) in each step's X can have grown at the end: an odd polynomial of a matrix
    moves by at most the largest divided difference of p over its (signed) singular values times the change."""
    S = np.concatenate([S, [0.0]])
    steps = []
    for a, b, c in coefficients:
        s = np.concatenate([S, -S])
        p = a * s + b * s ** 3 + c * s ** 5
        x, y = s[:, None], s[None, :]
        # (p(x) - p(y)) / (x - y), written out
        steps.append((np.abs(a + b * (x * x + x * y + y * y) + c * (x ** 4 + x ** 3 * y + x * x * y * y + x * y ** 3 + y ** 4)).max(),
                      np.linalg.norm(S)))
        S = a * S + b * S ** 3 + c * S ** 5
    total, grow = 0.0, 1.0
    for amp, size in reversed(steps):
        grow *= max(1.0, amp)
        total += grow * max(1.0, size)
    return total, np.linalg.norm(S)


def _check_orth(eng, M, dtype, coefficients=None, eps=1e-7):
    x = torch.from_numpy(M).to(dtype)
    M = x.double().numpy()
    coefs = [NS] * 5 if coefficients is None else coefficients
    got = eng.orthogonalise(x.cuda(), **({} if coefficients is None else dict(coefficients=coefficients)), eps=eps)
    assert got.dtype == dtype and got.shape == x.shape
    got, want = got.double().cpu().numpy(), sn.orthogonalise(M, coefs, eps)
    flat, g, w = M.reshape(-1, *M.shape[-2:]), got.reshape(-1, *M.shape[-2:]), want.reshape(-1, *M.shape[-2:])
    # what a step works with: 64 bits; else products of numbers held in 22 bits, summed in 32 over at most max(rows, cols) terms
    # (errors of random sign: the root of that, times 4)
    inner = 2.0 ** -52 if dtype == torch.float64 else 2.0 ** -22
    inner *= 8 * (1 + 4 * np.sqrt(max(M.shape[-2:])) / 8)
    u = _u(dtype)
    for m, a, b in zip(flat, g, w):
        grown, size = _amplified(np.linalg.svd(m, compute_uv=False) / (np.linalg.norm(m) + eps), coefs)
        off = np.linalg.norm(a - b)
        assert np.isfinite(off) and off <= inner * grown + u * np.linalg.norm(b) + 1e-30, (m.shape, off, inner * grown, size)


ORTH = [(1, 1, 1), (3, 1, 7), (2, 7, 1), (5, 10, 10), (2, 16, 40), (1, 64, 64), (2, 33, 65), (1, 65, 33), (1, 100, 100), (2, 128, 200),
        (1, 257, 130), (1, 130, 515)]


@pytest.mark.parametrize("dtype", [torch.float64, torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("shape", ORTH, ids=str)
def test_orthogonalise(eng, shape, dtype):
    rng = np.random.default_rng(30)
    _check_orth(eng, 1e-2 * rng.standard_normal(shape), dtype)


@pytest.mark.parametrize("shape", [(2, 100, 1501), (1, 1300, 66), (3, 150, 290), (1, 65, 4000)], ids=str)
def test_orthogonalise_in_64_bits(eng, shape):
    """Tiled products, the sums over a long side cut into parts."""
    rng = np.random.default_rng(79)
    _check_orth(eng, rng.standard_normal(shape), torch.float64)


@pytest.mark.parametrize("dtype", [torch.float64, torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("shape", [(9, 24, 100), (2, 10, 300), (2, 100, 40), (3, 64, 250), (2, 70, 400), (2, 480, 32), (3, 80, 150), (2, 17, 17)], ids=str)
def test_orthogonalise_on_chip(eng, shape, dtype):
    rng = np.random.default_rng(78)
    _check_orth(eng, rng.standard_normal(shape), dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("shape", [(523, 100, 120), (530, 140, 70)], ids=str)
def test_orthogonalise_a_few_tiles_over(eng, shape, dtype):
    """More tiles than the card takes at once, and a few: those are cut in four."""
    rng = np.random.default_rng(77)
    _check_orth(eng, rng.standard_normal(shape), dtype)


@pytest.mark.parametrize("dtype", [torch.float64, torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("shape", [(2, 12, 20), (1, 140, 90), (1, 96, 300)], ids=str)
def test_orthogonalise_of_low_rank(eng, shape, dtype):
    rng = np.random.default_rng(31)
    n, r, c = shape
    _check_orth(eng, rng.standard_normal((n, r, 3)) @ rng.standard_normal((n, 3, c)), dtype)


@pytest.mark.parametrize("size", [1e-30, 1e-12, 1e25])
@pytest.mark.parametrize("shape", [(2, 9, 14), (1, 80, 70)], ids=str)
def test_orthogonalise_of_any_scale(eng, shape, size):
    """The norm is taken in 64 bits: neither tiny nor huge entries lose it (eps is absolute, and 0 here)."""
    rng = np.random.default_rng(32)
    for dtype in (torch.float32, torch.bfloat16):
        _check_orth(eng, size * rng.standard_normal(shape), dtype, eps=0.0)


@pytest.mark.parametrize("shape", [(2, 9, 14), (1, 80, 70)], ids=str)
def test_orthogonalise_other_coefficients(eng, shape):
    rng = np.random.default_rng(33)
    M = rng.standard_normal(shape)
    _check_orth(eng, M, torch.float32, [(1.5, -0.5, 0.0)] * 16)
    _check_orth(eng, M, torch.float64, [(1.5, -0.5, 0.0)] * 16)
    _check_orth(eng, M, torch.float32, [NS, (15 / 8, -10 / 8, 3 / 8), (1.0, 0.0, 0.0)])
    # to the end: the convergent cubic's fixed point is the orthogonal factor itself
    X = eng.orthogonalise(torch.from_numpy(M).cuda(), coefficients=[(1.5, -0.5, 0.0)] * 16, eps=0.0).cpu().numpy()
    U, _, Vh = np.linalg.svd(M, full_matrices=False)
    np.testing.assert_allclose(X, U @ Vh, atol=1e-6)


@pytest.mark.parametrize("dtype", [torch.float64, torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("shape", [(2, 9, 14), (2, 70, 60), (2, 150, 200), (1, 300, 130)], ids=str)
def test_orthogonalise_with_steps_that_come_close_to_two(eng, shape, dtype):
    """One singular value where the first step carries it to 1.992 (0.3763), and a last step at 1.99 throughout."""
    from test_sequence import OPTIMISED

    rng = np.random.default_rng(85)
    n, r, c = shape
    d = min(r, c)
    S = np.abs(rng.standard_normal((n, d))) + 0.1
    S[:, 0] = 0.3763 / np.sqrt(1 - 0.3763 ** 2) * np.linalg.norm(S[:, 1:], axis=-1)
    U, V = (np.linalg.qr(rng.standard_normal((n, x, d)))[0] for x in (r, c))
    M = (U * S[:, None]) @ np.swapaxes(V, -1, -2)
    _check_orth(eng, M, dtype, OPTIMISED)
    _check_orth(eng, M, dtype, OPTIMISED + [(1.99, 0.0, 0.0)])


def test_orthogonalise_zeros_and_not_a_number(eng):
    for shape in ((3, 8, 8), (3, 70, 80)):
        for dtype in (torch.float32, torch.bfloat16, torch.float64):
            M = torch.randn(shape, device="cuda", dtype=torch.float64).to(dtype)
            clean = eng.orthogonalise(M)
            M[1] = 0.0
            got = eng.orthogonalise(M)
            assert not got[1].any() and torch.equal(got[0], clean[0]) and torch.equal(got[2], clean[2])
            for bad in (float("nan"), float("inf")):
                M[1, 3, 2] = bad
                got = eng.orthogonalise(M)  # the matrix that holds it is lost, its neighbours are not
                assert torch.isnan(got[1]).all() and torch.equal(got[0], clean[0]) and torch.equal(got[2], clean[2])


@pytest.mark.parametrize("dtype", [torch.float64, torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("shape", [(2, 10, 14), (2, 70, 60), (2, 150, 200), (1, 210, 130)], ids=str)
@pytest.mark.parametrize("rho", [1e-2, 1e-4, 1e-7, 1e-15, 1e-28])
def test_orthogonalise_far_below_eps(eng, shape, dtype, rho):
    """|M|_F much smaller than eps: X starts at |M| / eps and every step still works on it to its own precision, not to that of 1.

    A step's products are held in 22 bits (64-bit data: 52), and an error of that size relative to X leaves a step at most as large,
    relative to what X has become, as the largest over the smallest growth of a singular value in it.  All of them are below 485 rho, so
    that ratio is (1 + O((485 rho)^2)) for rho <= 1e-4, and for 1e-2 at most the product of the steps' ratios, computed below.  (bf16
    products take hi parts, 2^-11, of B X alone, whose size relative to a X is computed too.)"""
    rng = np.random.default_rng(81)
    eps = 1.0
    M = rng.standard_normal(shape)
    M *= rho / np.linalg.norm(M, axis=(-2, -1), keepdims=True)
    if dtype == torch.float16 and rho < 1e-3:
        M, eps = M * 2.0 ** 20, 2.0 ** 20  # (its smallest numbers are 6e-8)
    x = torch.from_numpy(M).to(dtype)
    M = x.double().numpy()
    # the result is about 485 rho for |X| = 1 spread over the matrix: well inside the normal numbers of all types here but fp16
    got, want = eng.orthogonalise(x.cuda(), eps=eps), sn.orthogonalise(M, [NS] * 5, eps)
    assert got.dtype == dtype
    got = got.double().cpu().numpy()
    for m, a, b in zip(M, got, want):
        S = np.linalg.svd(m, compute_uv=False) / (np.linalg.norm(m) + eps)
        total, ratio = 0.0, 1.0
        for c0, c1, c2 in [NS] * 5:
            gain = np.abs(c0 + c1 * S ** 2 + c2 * S ** 4)
            extra = np.abs(c1 * S ** 2 + c2 * S ** 4).max()
            S = gain * S
            ratio *= max(1.0, gain.max() / gain.min())
            unit = 2.0 ** -52 if dtype == torch.float64 else 2.0 ** -22
            total += 8 * unit * (1 + np.sqrt(max(m.shape)) / 2) + (2.0 ** -11 * extra / gain.min() if dtype == torch.bfloat16 else 0.0)
        size = np.linalg.norm(b)
        # (a result below the type's normal numbers: half of its smallest step for each entry)
        bound = (_u(dtype) + ratio * total) * size + _least(dtype) * np.sqrt(b.size)
        assert np.linalg.norm(a - b) <= bound, (np.linalg.norm(a - b) / size, bound / size)


@pytest.mark.parametrize("dtype", [torch.float64, torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("shape", [(3, 150, 200), (3, 210, 100)], ids=str)
def test_orthogonalise_zeros_and_not_a_number_in_tiles(eng, shape, dtype):
    """The tiled products keep the matrices of a batch apart as the others do."""
    M = torch.from_numpy(np.random.default_rng(82).standard_normal(shape)).to(dtype).cuda()
    clean = eng.orthogonalise(M)
    M[1] = 0.0
    got = eng.orthogonalise(M)
    assert not got[1].any() and torch.equal(got[0], clean[0]) and torch.equal(got[2], clean[2])
    for bad in (float("nan"), float("inf")):
        M[1, 3, 2] = bad
        got = eng.orthogonalise(M)
        assert torch.isnan(got[1]).all() and torch.equal(got[0], clean[0]) and torch.equal(got[2], clean[2])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("shape", [(90, 200, 260), (90, 260, 200), (172, 200, 260), (172, 260, 200), (1, 600, 700)], ids=str)
def test_orthogonalise_in_tiles_off_the_diagonal(eng, shape, dtype):
    """Enough matrices for tiles of 128, with several of them along each side: off the diagonal, stored with their mirror image; 172: the
    last few of 516 (A, B) and 1032 (X) cut in four, off the diagonal too.  (1, 600, 700): tiles of 64 in bands of 8, the last partial."""
    _check_orth(eng, np.random.default_rng(83).standard_normal(shape), dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_orthogonalise_in_several_bands_of_large_tiles(eng, dtype):
    """9 x 11 tiles of 128 for each of 6 matrices: a second band of one tile."""
    _check_orth(eng, np.random.default_rng(84).standard_normal((6, 1100, 1290)), dtype)


def test_orthogonalise_views_and_leading_axes(eng):
    M = torch.randn(2, 3, 20, 12, device="cuda")
    want = eng.orthogonalise(M)
    assert torch.equal(eng.orthogonalise(M.transpose(-1, -2).contiguous().transpose(-1, -2)), want)
    assert torch.equal(eng.orthogonalise(M[1, 2]), want[1, 2])
    assert torch.equal(eng.orthogonalise(M.cpu().numpy()), want)


# ------------------------------------------------------------------------------- together, streams, graphs, other callers
def test_a_training_step_of_a_state_space_layer(eng):
    """x -> q, k, v by weights, the recurrence, a quadratic loss; its gradient by the kernels, the weights' update orthogonalised;
    against the same step in 64 bits."""
    rng = np.random.default_rng(40)
    B, T, H, D, N = 2, 70, 2, 16, 24
    x = rng.standard_normal((B, T, N))
    W = {n: 0.3 * rng.standard_normal((N, H * D)) for n in "qkv"}
    g = -rng.random(H) * 0.2
    y = rng.standard_normal((B, T, H, D))
    p = {n: (x @ W[n]).reshape(B, T, H, D) for n in "qkv"}
    o, _ = sn.attention(p["q"], p["k"], p["v"], g, 0.25)
    grad = sn.attention_gradient(p["q"], p["k"], p["v"], g, o - y, 0.25)
    xd, gd, yd = _dev(x), _dev(g), _dev(y)
    pd = {n: (xd @ _dev(W[n])).view(B, T, H, D) for n in "qkv"}
    od, _ = eng.linear_attention(pd["q"], pd["k"], pd["v"], gd, scale=0.25)
    gr = eng.linear_attention_backward(pd["q"], pd["k"], pd["v"], gd, od - yd, scale=0.25)
    # in 32 bits: sums of at most T terms, in the gradients of products of three sums
    assert float((od.double().cpu() - torch.from_numpy(o)).norm()) < 1e-5 * np.linalg.norm(o)
    np.testing.assert_allclose(gr["log_decay"].cpu().numpy(), grad["log_decay"], rtol=1e-4)
    for n in "qkv":
        dW = np.einsum("btn,btm->nm", x, grad[n].reshape(B, T, -1))
        dWd = xd.reshape(-1, N).T @ gr[n].reshape(B * T, -1)
        assert float((dWd.double().cpu() - torch.from_numpy(dW)).norm()) < 2e-5 * np.linalg.norm(dW)
        up, upd = sn.orthogonalise(dW, [NS] * 5), eng.orthogonalise(dWd)
        # an error in dW grows by at most a^5 = 485 on its way through five steps
        assert np.linalg.norm(upd.double().cpu().numpy() - up) < 485 * 2e-5


def test_the_update_of_a_filters_transition_matrices(eng):
    """value_and_grad's gradient of T, one matrix for each draw, straight into the update."""
    import workloads as W

    w = W.structural(B=8, n=40)
    _, _, g = eng.value_and_grad(w["y"], w["a0"], w["P0"], w["T"], w["Z"], w["R"], w["H"], w["Q"])
    got = eng.orthogonalise(g["T"])
    assert got.dtype == torch.float64 and got.shape == g["T"].shape
    np.testing.assert_allclose(got.cpu().numpy(), sn.orthogonalise(g["T"].cpu().numpy(), [NS] * 5), atol=1e-9)


def _everything(eng, t):
    """One call of each operator on tensors of `t`."""
    o, s = eng.linear_attention(t["q"], t["k"], t["v"], t["g"])
    d = eng.linear_attention_backward(t["q"], t["k"], t["v"], t["g"], t["v"], initial_state=s)
    out = s.clone()
    o1, _ = eng.linear_attention_step(t["q"][:, 0], t["k"][:, 0], t["v"][:, 0], t["g"][:, 0], s, state_out=out)
    return [o, s, d["q"], d["k"], d["v"], d["log_decay"], d["initial_state"], o1, out, eng.orthogonalise(t["M"]), eng.orthogonalise(t["M"][:, :9, :9])]


def _tensors(seed, dtype):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    return dict(q=r(2, 150, 1, 32).to(dtype), k=r(2, 150, 1, 32).to(dtype), v=r(2, 150, 2, 48).to(dtype), g=-r(2, 150, 2).abs(), M=r(2, 90, 130).to(dtype))


def test_on_another_stream(eng):
    t = _tensors(1, torch.bfloat16)
    want = _everything(eng, t)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _everything(eng, t)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", list(TYPES))
def test_two_captured_graphs(eng, dtype):
    """Captured, replayed several times with new inputs in place and eager work between, on two streams at once."""
    sets = [_tensors(s, TYPES[dtype]) for s in (2, 3)]
    graphs, outs = [], []
    for t in sets:
        _everything(eng, t)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_everything(eng, t))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for round_ in range(4):
        fresh = [_tensors(10 * round_ + s, TYPES[dtype]) for s in (4, 5)]
        want = []
        for t, f in zip(sets, fresh):
            for n in t:
                t[n].copy_(f[n])
            want.append(_everything(eng, t))
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for have, w in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(have, w)), round_


def test_inputs_that_autograd_watches_and_host_arrays(eng):
    t = _tensors(6, torch.float32)
    want = _everything(eng, t)
    w = {n: x.clone().requires_grad_() for n, x in t.items()}
    got = _everything(eng, w)
    assert all(torch.equal(a, b) and not a.requires_grad for a, b in zip(got, want))
    host = {n: x.cpu().numpy() for n, x in t.items()}
    o, s = eng.linear_attention(host["q"], host["k"], host["v"], host["g"])
    assert torch.equal(o, want[0]) and torch.equal(s, want[1])
