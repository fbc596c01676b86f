"""Attention in float64 with the error that the kernels' arithmetic allows, for the operator tests.

The kernels take 16-bit (or fp32) inputs exactly, form scores and sums in fp32, and round the result
once. For one query row with visible keys j, s_j = scale q.k_j, p = softmax(s), out = sum_j p_j v_j:

  * a score is a sum of d exact products in fp32, times scale * log2(e) (two more roundings):
    |ds_j| <= delta = 2^-24 ((d + 8) scale sum_i |q_i k_ji| + 4 |s_j|); exp2 adds 2^-22 relative;
  * a relative change of every p_j by at most r moves the normalised weights by at most 2 r, so the
    output by at most 2 r sum_j p_j |v_j|; r = delta + 2^-21;
  * the weights are multiplied with the values as `p_bits`-bit numbers: relative error 2^-p_bits. A bf16
    has 8 significant bits, so rounding to nearest is off by half a step = torch.finfo.eps / 2 = 2^-8 of
    the value (fp16 11 bits: 2^-11); two parts square that. fp16 has no steps below 2^-24, so a weight
    is off by up to 2^-25 there as well; the weights are relative to a running maximum that was a
    score's own value once, so their sum l >= 1 and each key adds at most 2^-25 |v_j|;
  * the sums over n keys run in fp32: 16 keys an instruction, so n / 16 + 64 roundings of 2^-24, twice;
  * one rounding to the output type: half a step.
"""
import torch

# significant bits of a weight as the product with V sees it
P_SPLIT = {torch.bfloat16: 16, torch.float16: 22, torch.float32: 24}  # two 16-bit parts (decode kernel)
P_SINGLE = {torch.bfloat16: 8, torch.float16: 11, torch.float32: 24}  # one 16-bit number, rounded to nearest


def attend64(q, k, v, scale, seen=None, p_bits=None):
    """q [..., r, d], k, v [..., n, d], seen (broadcastable to [..., r, n]) True where visible. Returns
    (out float64, tolerance without the output rounding's dependence on itself) for outputs of q's
    dtype; rows that see nothing give zeros and tolerance 0."""
    p_bits = P_SINGLE[q.dtype] if p_bits is None else p_bits
    dt, d, n = q.dtype, q.shape[-1], k.shape[-2]
    q, k, v = q.double(), k.double(), v.double()
    x = (q @ k.transpose(-1, -2)) * scale
    size = (q.abs() @ k.abs().transpose(-1, -2)) * abs(scale) * (d + 8) + 4 * x.abs()
    if seen is None:
        seen = torch.ones_like(x, dtype=torch.bool)
    seen = seen.expand(x.shape)
    x = x.masked_fill(~seen, -float("inf"))
    empty = ~seen.any(-1, keepdim=True)
    p = torch.softmax(x.masked_fill(empty, 0.0), -1).masked_fill(empty, 0.0)
    v0 = v.masked_fill(~seen.any(-2).unsqueeze(-1), 0.0)  # what no row sees may hold anything
    out = p @ v0
    delta = 2.0 ** -24 * size.masked_fill(~seen, 0.0).nan_to_num(0.0).amax(-1, keepdim=True) if n else 0.0
    rel = 2 * (delta + 2.0 ** -21) + 2.0 ** -p_bits + (n / 16 + 64) * 2.0 ** -23
    tol = rel * (p @ v0.abs())
    if dt == torch.float16:
        tol = tol + 2.0 ** -25 * (seen.double() @ v0.abs())
    half = torch.finfo(dt).eps / 2
    tiny = 2.0 ** -25 if dt == torch.float16 else 0.0
    return out, tol * (1 + half) + half * out.abs() + tiny * (~empty)


def assert_within(got, ref, tol):
    err = (got.double() - ref).abs()
    assert torch.isfinite(got).all(), "not finite"
    assert (err <= tol).all(), f"max error {float(err.max()):.3g}, worst excess {float((err - tol).max()):.3g}"
