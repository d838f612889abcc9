"""The operators of ssm_ops.py restated token by token on float64 tensors, differentiable by torch: test infrastructure."""
import torch
import torch.nn.functional as F


def causal_conv(x, weight, bias=None, silu=True, initial_state=None, lengths=None):
    """(y, final state) of x [batch, length, channels]; padding is cut off before anything is computed."""
    B, L, D = x.shape
    W = weight.shape[1]
    ys, states = [], []
    for b in range(B):
        n = L if lengths is None else min(max(int(lengths[b]), 0), L)
        first = x.new_zeros(W - 1, D) if initial_state is None else initial_state[b]
        rows = torch.cat([first, x[b, :n]])
        y = []
        for t in range(n):
            pre = (weight.t() * rows[t:t + W]).sum(0)
            if bias is not None:
                pre = pre + bias
            y.append(F.silu(pre) if silu else pre)
        y = torch.stack(y) if y else x.new_zeros(0, D)
        ys.append(torch.cat([y, x.new_zeros(L - n, D)]))
        states.append(rows[n:])
    return torch.stack(ys), torch.stack(states)


def selective_scan(u, dt, A, B, C, D=None, z=None, dt_bias=None, softplus=True, initial_state=None, lengths=None):
    """(y, final state) with B, C [batch, length, groups, states]."""
    nb, L, ch = u.shape
    N, G = A.shape[1], B.shape[2]
    ys, states = [], []
    for b in range(nb):
        n = L if lengths is None else min(max(int(lengths[b]), 0), L)
        h = u.new_zeros(ch, N) if initial_state is None else initial_state[b]
        raw = dt[b, :n] if dt_bias is None else dt[b, :n] + dt_bias
        delta = F.softplus(raw, threshold=1e9) if softplus else raw
        y = []
        for t in range(n):
            Bt, Ct = (m[b, t].repeat_interleave(ch // G, 0) for m in (B, C))
            h = torch.exp(delta[t, :, None] * A) * h + (delta[t] * u[b, t])[:, None] * Bt
            o = (h * Ct).sum(-1)
            if D is not None:
                o = o + D * u[b, t]
            y.append(o * F.silu(z[b, t]) if z is not None else o)
        y = torch.stack(y) if y else u.new_zeros(0, ch)
        ys.append(torch.cat([y, u.new_zeros(L - n, ch)]))
        states.append(h)
    return torch.stack(ys), torch.stack(states)


def block_norm(h, y, w1, w2, gate=None, scale=None, eps=1e-6):
    def norm(v, w):
        return w * v / torch.sqrt(v.pow(2).mean(-1, keepdim=True) + eps)
    p = norm(y, w1)
    if gate is not None:
        p = p * torch.sigmoid(gate)
    if scale is not None:
        p = p * scale
    out = h + p
    return out, norm(out, w2)
