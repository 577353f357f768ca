"""CPU restatement, in 64 bits, of the 8-bit KV cache: a row is 128 e4m3
values and an exponent byte, standing for e4m3 * 2^(byte - 127)."""

from __future__ import annotations

import math

import torch

MIN_EXP, MAX_EXP = -117, 119
E4M3_MAX = 448.0


def e4m3_value(code: int) -> float:
    """The number an e4m3 code stands for (bias 7, 3 fraction bits, no infinities)."""
    sign = -1.0 if code & 0x80 else 1.0
    e, m = (code >> 3) & 15, code & 7
    if e == 15 and m == 7:
        return math.nan
    return sign * (math.ldexp(8 + m, e - 10) if e else math.ldexp(m, -9))


E4M3 = torch.tensor([e4m3_value(c) for c in range(256)], dtype=torch.float64)


def row_exponent(top: float) -> int:
    """The smallest k in [MIN_EXP, MAX_EXP] with top <= 448 * 2^k (MAX_EXP if none)."""
    k = MIN_EXP
    while k < MAX_EXP and top > math.ldexp(E4M3_MAX, k):
        k += 1
    return k


def quantise_ref(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows [..., 128] to (codes uint8 [..., 128], exponent bytes uint8 [...])."""
    v = x.double()
    flat = v.reshape(-1, v.shape[-1])
    codes = torch.empty(flat.shape, dtype=torch.uint8)
    exps = torch.empty(flat.shape[0], dtype=torch.uint8)
    grid = E4M3[:127]
    for i, row in enumerate(flat):
        fin = row[torch.isfinite(row)].abs()
        k = row_exponent(float(fin.max()) if fin.numel() else 0.0)
        y = torch.nan_to_num(row.abs() * math.ldexp(1.0, -k), nan=0.0, posinf=E4M3_MAX)
        y = y.clamp(max=E4M3_MAX)
        hi = torch.searchsorted(grid, y).clamp(1, 126)
        up, down = grid[hi] - y, y - grid[hi - 1]
        c = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, hi - 1)
        c = torch.where(torch.isnan(row), torch.full_like(c, 127), c + 128 * torch.signbit(row).long())
        codes[i] = c.to(torch.uint8)
        exps[i] = k + 127
    return codes.reshape(v.shape), exps.reshape(v.shape[:-1])


def _two(k: torch.Tensor) -> torch.Tensor:
    """2^k in 64 bits, from its exponent field."""
    return ((k.long() + 1023) << 52).view(torch.float64)


def dequantise_ref(codes: torch.Tensor, exps: torch.Tensor) -> torch.Tensor:
    """Codes [..., 128] and exponent bytes [...] to 64-bit values."""
    return E4M3.to(codes.device)[codes.long()] * _two(exps.long() - 127).unsqueeze(-1)


def store_fp8_ref(key, value, k_codes, v_codes, k_exp, v_exp, slots) -> None:
    """In place on codes [blocks, block, Hk, 128] and bytes [blocks, Hk, block]."""
    block = k_codes.shape[1]
    kq, vq = quantise_ref(key), quantise_ref(value)
    for i, s in enumerate(slots.tolist()):
        if s < 0 or s >= k_codes.shape[0] * block:
            continue
        for codes, exps, (q, e) in ((k_codes, k_exp, kq), (v_codes, v_exp, vq)):
            codes[s // block, s % block] = q[i]
            exps[s // block, :, s % block] = e[i]


def sequence_ref(codes, exps, table, length) -> torch.Tensor:
    """Rows [length, Hk, 128] of one sequence, 64-bit."""
    block = codes.shape[1]
    pages = table[:-(-length // block)].long()
    x = dequantise_ref(codes[pages], exps[pages].transpose(1, 2))
    return x.reshape(-1, *x.shape[2:])[:length]


def decode_fp8_ref(q, k_codes, v_codes, k_exp, v_exp, tables, lens, scale):
    """(out, bound) in 64 bits: attention of one token per row, and how far a
    result in bf16 may be from it.

    The bound counts, with A = sum_j p_j |V_j| (elementwise):
      * the result's rounding to bf16: 2^-8 |out|;
      * the weights' rounding to 11 bits (f16) before the product with V:
        2^-11 A;
      * the scores' error in 32 bits: a sum of 128 products, then a product
        with the scale, is off by at most 130 * 2^-24 * sum_i |q_i K_ji| *
        scale for token j; e = the largest of these; a weight p_j and the
        weights' sum are each off by a factor within e^(+-e): 2 e (A + |out|)
        (with |out| <= A: 4 e A);
      * exp2 in hardware and the 32-bit sums of the weights and of the
        products over the tokens, 2^-22 each and one rounding per 16 tokens:
        (2^-20 + len / 16 * 2^-24) * A;
      * underflow: a weight below 2^-126 is 0 in 32 bits, which moves the
        result by at most 2^-126 |V_j| for each token; a product weight
        w_j = p_j * 2^k_j (k_j the row's exponent) held in f16 as 2^15 times
        its share of the largest, W, has the absolute error 2^-40 W where it is
        below 2^-29 W (f16's normal numbers begin at 2^-14 and its subnormal
        step is 2^-24: half of it, over 2^15), which moves the result by
        2^-40 W |code_j| for each such token.
    """
    B, Hq, D = q.shape
    Hk = k_codes.shape[2]
    g = Hq // Hk
    out = torch.zeros(B, Hq, D, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    for b, n in enumerate(lens.tolist()):
        if n == 0:
            continue
        k = sequence_ref(k_codes, k_exp, tables[b], n)
        v = sequence_ref(v_codes, v_exp, tables[b], n)
        for h in range(Hk):
            qq = q[b, h * g:(h + 1) * g].double()
            p = torch.softmax(qq @ k[:, h].T * scale, -1)
            at = tables[b, torch.arange(n, device=q.device) // v_codes.shape[1]].long()
            byte = v_exp[at, h, torch.arange(n, device=q.device) % v_codes.shape[1]].long()
            two_k = _two(byte - 127)
            w = p * two_k
            top = w.amax(-1, keepdim=True)
            small = torch.where(w < 2.0 ** -29 * top, 2.0 ** -40 * top, 0.0)
            under = small @ (v[:, h].abs() / two_k.unsqueeze(1)) + 2.0 ** -126 * v[:, h].abs().sum(0)
            e = 130 * 2.0 ** -24 * float((qq.abs() @ k[:, h].abs().T).amax()) * scale
            o = p @ v[:, h]
            a = p @ v[:, h].abs()
            out[b, h * g:(h + 1) * g] = o
            bound[b, h * g:(h + 1) * g] = 2.0 ** -8 * o.abs() + under + a * (
                2.0 ** -11 + 4 * e + 2.0 ** -20 + n / 16 * 2.0 ** -24)
    return out, bound
