"""The recurrence of ``sequence_numpy`` and its gradient, in 64 bits and one token at a time, for whole batches of many heads at once
(torch, on the device of its inputs): the same arguments and results, fast enough for sequences that are cut into many chunks."""
import numpy as np
import torch


def _operands(q, k, v, log_decay, s0, lengths, device):
    q, k, v, g = (torch.as_tensor(np.array(x), dtype=torch.float64, device=device) for x in (q, k, v, log_decay))
    B, T, H, V = v.shape
    per = H // q.shape[2]
    q, k = q.repeat_interleave(per, 2), k.repeat_interleave(per, 2)
    live = torch.ones(B, T, dtype=torch.bool, device=device)
    if lengths is not None:
        live = torch.arange(T, device=device)[None] < torch.as_tensor(np.asarray(lengths), device=device)[:, None]
    a = g.expand(B, T, H).exp()
    S = torch.zeros(B, H, q.shape[-1], V, dtype=torch.float64, device=device)
    if s0 is not None:
        S = torch.as_tensor(np.asarray(s0), dtype=torch.float64, device=device).clone()
    return q, k, v, a, S, live


def _states(k, v, a, S, live):
    """S before the first token and behind every token (a token that is not live leaves it as it is)."""
    out = [S]
    for t in range(k.shape[1]):
        new = a[:, t, :, None, None] * S + k[:, t, :, :, None] * v[:, t, :, None, :]
        S = torch.where(live[:, t, None, None, None], new, S)
        out.append(S)
    return out


def attention(q, k, v, log_decay, scale, s0=None, lengths=None, device="cpu"):
    q, k, v, a, S, live = _operands(q, k, v, log_decay, s0, lengths, device)
    S = _states(k, v, a, S, live)
    o = torch.stack([scale * (q[:, t, :, :, None] * S[t + 1]).sum(-2) for t in range(q.shape[1])], 1)
    return (o * live[:, :, None, None]).cpu().numpy(), S[-1].cpu().numpy()


def attention_gradient(q, k, v, log_decay, g_o, scale, s0=None, lengths=None, g_sT=None, device="cpu"):
    G, per_token = np.shape(q)[2], np.ndim(log_decay) > 1
    q, k, v, a, S, live = _operands(q, k, v, log_decay, s0, lengths, device)
    go = torch.as_tensor(np.asarray(g_o), dtype=torch.float64, device=device)
    B, T, H, V = v.shape
    S = _states(k, v, a, S, live)
    R = torch.zeros_like(S[0]) if g_sT is None else torch.as_tensor(np.asarray(g_sT), dtype=torch.float64, device=device).clone()
    dq, dk, dv, dg = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v), torch.zeros_like(a)
    for t in reversed(range(T)):
        on = live[:, t, None, None]
        at = R + scale * q[:, t, :, :, None] * go[:, t, :, None, :]
        dq[:, t] = scale * (S[t + 1] * go[:, t, :, None, :]).sum(-1) * on
        dk[:, t] = (at * v[:, t, :, None, :]).sum(-1) * on
        dv[:, t] = (at * k[:, t, :, :, None]).sum(-2) * on
        at = a[:, t, :, None, None] * at
        dg[:, t] = (at * S[t]).sum((-2, -1)) * on[..., 0]
        R = torch.where(on[..., None], at, R)
    dq, dk = (x.unflatten(2, (G, H // G)).sum(3) for x in (dq, dk))
    out = dict(q=dq, k=dk, v=dv, log_decay=dg if per_token else dg.sum((0, 1)), initial_state=R)
    return {n: x.cpu().numpy() for n, x in out.items()}
