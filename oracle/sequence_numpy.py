"""The sequence operators from their definitions, in 64 bits and one token at a time (numpy)."""
import numpy as np


def attention(q, k, v, log_decay, scale, s0=None, lengths=None):
    """S_t = exp(log_decay_t) S_{t-1} + k_t v_t', o_t = scale S_t' q_t -> (o (B,T,H,V), S (B,H,K,V))."""
    q, k, v, a = _heads(q, k, v, log_decay)
    B, T, H, V = v.shape
    S = np.zeros((B, H, q.shape[-1], V)) if s0 is None else np.array(s0, dtype=np.float64)
    o = np.zeros((B, T, H, V))
    for b in range(B):
        for t in range(_length(lengths, b, T)):
            S[b] = a[b, t][:, None, None] * S[b] + k[b, t][:, :, None] * v[b, t][:, None, :]
            o[b, t] = scale * np.einsum("hk,hkv->hv", q[b, t], S[b])
    return o, S


def attention_gradient(q, k, v, log_decay, g_o, scale, s0=None, lengths=None, g_sT=None):
    """Gradient of <g_o, o> + <g_sT, S_T>: dict of q, k, v, log_decay, initial_state, from R_t = dL/dS_t."""
    G, per_token = np.shape(q)[2], np.ndim(log_decay) > 1
    q, k, v, a = _heads(q, k, v, log_decay)
    go = np.asarray(g_o, dtype=np.float64)
    B, T, H, V = v.shape
    K = q.shape[-1]
    dq, dk, dv, dg = np.zeros_like(q), np.zeros_like(k), np.zeros_like(v), np.zeros((B, T, H))
    ds0 = np.zeros((B, H, K, V))
    for b in range(B):
        n = _length(lengths, b, T)
        before = [np.zeros((H, K, V)) if s0 is None else np.array(s0[b], dtype=np.float64)]
        for t in range(n):
            before.append(a[b, t][:, None, None] * before[-1] + k[b, t][:, :, None] * v[b, t][:, None, :])
            dq[b, t] = scale * np.einsum("hkv,hv->hk", before[-1], go[b, t])
        R = np.zeros((H, K, V)) if g_sT is None else np.array(g_sT[b], dtype=np.float64)
        for t in reversed(range(n)):
            R = R + scale * q[b, t][:, :, None] * go[b, t][:, None, :]
            dk[b, t] = np.einsum("hkv,hv->hk", R, v[b, t])
            dv[b, t] = np.einsum("hkv,hk->hv", R, k[b, t])
            R = a[b, t][:, None, None] * R
            dg[b, t] = np.sum(R * before[t], axis=(-2, -1))
        ds0[b] = R
    dq, dk = (x.reshape(B, T, G, H // G, K).sum(3) for x in (dq, dk))
    return dict(q=dq, k=dk, v=dv, log_decay=dg if per_token else dg.sum((0, 1)), initial_state=ds0)


def attention_step(q, k, v, log_decay, state, scale, slots=None):
    """One token for each row, rows in order -> (o (B,H,V), pool)."""
    pool = np.array(state, dtype=np.float64)
    B = np.shape(v)[0]
    o = np.zeros(np.shape(v))
    for b in range(B):
        at = b if slots is None else int(slots[b])
        if 0 <= at < pool.shape[0]:
            g = log_decay if np.ndim(log_decay) == 1 else np.asarray(log_decay)[b:b + 1, None]
            ob, S = attention(q[b:b + 1, None], k[b:b + 1, None], v[b:b + 1, None], g, scale, pool[at][None])
            o[b], pool[at] = ob[0, 0], S[0]
    return o, pool


def orthogonalise(M, coefficients, eps=1e-7):
    X = np.asarray(M, dtype=np.float64)
    tall = X.shape[-2] > X.shape[-1]
    if tall:
        X = np.swapaxes(X, -1, -2)
    X = X / (np.sqrt(np.sum(X * X, axis=(-2, -1), keepdims=True)) + eps)
    for a, b, c in coefficients:
        A = X @ np.swapaxes(X, -1, -2)
        X = a * X + (b * A + c * (A @ A)) @ X
    return np.swapaxes(X, -1, -2) if tall else X


def _length(lengths, b, T):
    return T if lengths is None else min(max(int(lengths[b]), 0), T)


def _heads(q, k, v, log_decay):
    q, k, v = (np.asarray(x, dtype=np.float64) for x in (q, k, v))
    per = v.shape[2] // q.shape[2]
    a = np.exp(np.broadcast_to(np.asarray(log_decay, dtype=np.float64), v.shape[:3]))
    return np.repeat(q, per, 2), np.repeat(k, per, 2), v, a
