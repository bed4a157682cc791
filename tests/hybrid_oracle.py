"""Plain 64-bit implementations of the hybrid family's block operators, written from their definitions; they share no code with the package."""
import math

import torch

F64 = torch.float64


def gdn_rows(inp, first, rows, start_conv, start_rec, conv_w, ssm_a, dt_bias, norm_w, n_k, v_head_offset, eps, z_off, ab_off):
    """One sequence, row after row.  inp: bf16 rows; first / rows: its rows; start_*: state in front (None: zeros).  Returns out [rows, n_v d] and
    the states behind every row, [(conv, rec), ...]."""
    n_v, d, K = ssm_a.numel(), norm_w.numel(), conv_w.shape[1]
    C = (2 * n_k + n_v) * d
    win = torch.zeros(C, K - 1, dtype=F64) if start_conv is None else start_conv.to(F64)
    S = torch.zeros(n_v, d, d, dtype=F64) if start_rec is None else start_rec.to(F64).clone()
    w, a_, dt, g = conv_w.to(F64), ssm_a.to(F64), dt_bias.to(F64), norm_w.to(F64)
    out, states = torch.zeros(rows, n_v * d, dtype=F64), []
    for t in range(rows):
        x = inp[first + t].to(F64)
        full = torch.cat([win, x[:C, None]], 1)
        y = (full * w).sum(1)
        y = y / (1 + torch.exp(-y))
        win = full[:, 1:]
        for h in range(n_v):
            kh = (h + v_head_offset) % n_k
            q, k = y[kh * d:(kh + 1) * d], y[(n_k + kh) * d:(n_k + kh + 1) * d]
            v = y[(2 * n_k + h) * d:(2 * n_k + h + 1) * d]
            q = q / math.sqrt(float((q * q).sum()) + 1e-6) / math.sqrt(d)
            k = k / math.sqrt(float((k * k).sum()) + 1e-6)
            z = float(x[ab_off + h]) + float(dt[h])
            decay = math.exp(float(a_[h]) * (z if z > 40 else math.log1p(math.exp(z))))
            beta = 1 / (1 + math.exp(-float(x[ab_off + n_v + h])))
            M = decay * S[h]
            u = beta * (v - M.t() @ k)
            S[h] = M + torch.outer(k, u)
            o = S[h].t() @ q
            gate = x[z_off + h * d:z_off + (h + 1) * d]
            out[t, h * d:(h + 1) * d] = o / math.sqrt(float((o * o).mean()) + eps) * g * gate / (1 + torch.exp(-gate))
        states.append((win.clone(), S.clone()))
    return out, states


def rope_part(rows, n_heads, n_kv_heads, D, q_norm, k_norm, freqs, magnitude, positions, eps, gated, interleaved):
    """Rows -> (queries [T, H, D], keys [T, Hk, D], values [T, Hk, D])."""
    T, per = rows.shape[0], 2 if gated else 1
    x = rows.to(F64).reshape(T, n_heads * per + 2 * n_kv_heads, D)
    q, k, v = x[:, :n_heads * per:per], x[:, n_heads * per:n_heads * per + n_kv_heads], x[:, n_heads * per + n_kv_heads:]
    n = freqs.numel()

    def turn(h, gain):
        h = h.clone()
        if gain is not None:
            h = h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps) * gain.to(F64)
        out = h.clone()
        for t in range(T):
            for i in range(n):
                a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
                ang = float(positions[t]) * float(freqs[i])
                c, s = magnitude * math.cos(ang), magnitude * math.sin(ang)
                out[t, :, a] = h[t, :, a] * c - h[t, :, b] * s
                out[t, :, b] = h[t, :, b] * c + h[t, :, a] * s
        return out

    return turn(q, q_norm), turn(k, k_norm), v


def attention_rows(q, kv, table, seq_len, R, n_kv_heads, scale, gate=None):
    """The R rows of one sequence over its own table: q [R, H, D]; row r sees keys < seq_len - (R - 1 - r).  Returns the rows and, as large, sum p |v|."""
    H, D = q.shape[1:]
    out, size = torch.zeros(R, H, D, dtype=F64), torch.zeros(R, H, D, dtype=F64)
    for r in range(R):
        n = seq_len - (R - 1 - r)
        if n <= 0:
            continue
        pages = table[:(n + 63) // 64].long()
        for h in range(H):
            kvh = h // (H // n_kv_heads)
            K = kv[pages, 0, kvh].reshape(-1, D)[:n].to(F64)
            V = kv[pages, 1, kvh].reshape(-1, D)[:n].to(F64)
            p = torch.softmax(K @ q[r, h].to(F64) * scale, 0)
            out[r, h], size[r, h] = p @ V, p @ V.abs()
    g = 1.0 if gate is None else 1 / (1 + torch.exp(-gate.to(F64)))
    return out * g, size * g
