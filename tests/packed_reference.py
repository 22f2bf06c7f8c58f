"""Plain 64-bit reference of the packed-batch attention and the tolerance its
tests derive from the kernel's roundings."""

import torch

# bound on the relative error of the kernel's 2^x, far below the rounding of the
# weights to the input type that follows it
EXP_ERR = {torch.float16: 2.0 ** -17, torch.bfloat16: 2.0 ** -13}


def reference(query, q_lens, keys, values, scale, causal=True, prefix=None):
    """query [T, H_q, D]; keys/values: per sequence [n_b, H_kv, D]; prefix: (K, V) [H_kv, P, D].

    Returns (out, tol), both [T, H_q, D] in 64 bits.  With w the exact softmax weights and A = sum_j w_j |V_j|
    (per dim), the kernel's error is at most the sum of
      * A eps / 2: each weight is rounded to the input type (half a step);
      * |out| eps / 2 <= A eps / 2: the output's rounding;
      * 2 A (E_s + EXP_ERR + 2^-21): a relative error of the weights enters numerator and denominator; E_s is the
        absolute error of a score, (D + 4) 2^-23 scale sum_d |q_d k_jd| for fp32 sums of D exact products and the
        scaling, and 2^-21 covers the joins of pieces;
      * (n + 4) 2^-23 A: fp32 sums over n keys in the second product, and as much in the denominator
        (halved steps: 2^-24 each)."""
    T, Hq, D = query.shape
    dt = query.dtype
    out = torch.zeros((T, Hq, D), dtype=torch.float64, device=query.device)
    tol = torch.zeros_like(out)
    eps = torch.finfo(dt).eps
    t0 = 0
    for b, m in enumerate(q_lens):
        k, v = keys[b].double(), values[b].double()
        n_own, far = k.shape[0], 0
        if prefix is not None:
            far = prefix[0].shape[1]
            k = torch.cat((prefix[0].double().transpose(0, 1), k))
            v = torch.cat((prefix[1].double().transpose(0, 1), v))
        n, Hkv = k.shape[0], k.shape[1]
        G = Hq // Hkv
        if m and n:
            q = query[t0:t0 + m].double()
            seen = torch.ones((m, n), dtype=torch.bool, device=q.device)
            if causal:
                last = torch.arange(m, device=q.device) + (far + n_own - m)
                seen = torch.arange(n, device=q.device)[None] <= last[:, None]
                if far:
                    seen[:, :far] = True
            for h in range(Hq):
                kh, vh = k[:, h // G], v[:, h // G]
                s = q[:, h] @ kh.T * scale
                w = torch.softmax(s.masked_fill(~seen, float("-inf")), -1).nan_to_num_(0.0)
                a = w @ vh.abs()
                mag = (q[:, h].abs() @ kh.abs().T).masked_fill(~seen, 0.0).amax(-1, keepdim=True)
                e_s = (D + 4) * 2.0 ** -23 * scale * mag
                out[t0:t0 + m, h] = w @ vh
                tol[t0:t0 + m, h] = a * (eps + 2 * (e_s + EXP_ERR[dt] + 2.0 ** -21) + (n + 4) * 2.0 ** -23)
        t0 += m
    # results below the type's normal range round to its smallest step
    tol += torch.finfo(dt).smallest_normal * eps
    return out, tol


def lens_tensor(lens):
    c = [0]
    for n in lens:
        c.append(c[-1] + n)
    return torch.tensor(c, dtype=torch.int32, device="cuda")
