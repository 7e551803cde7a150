"""How far paged decode attention may be off when its weights are not rounded to
16 bits before the product with V (they enter as a 16-bit value and a 16-bit
remainder).  With p_j the weights relative to the largest (so that their sum is
at least 1), o the output, A = sum_j p_j |v_j| normalised and u the unit roundoff:

  u |o|          rounding the output (fp16: up to 2^-25 below its normal range);
  2 u^2 A        the remainder's own rounding: |p - hi| <= u p, and u of that; the
                 second one covers its 32-bit difference;
  2^-25 sum |v|  fp16 only: a remainder below the normal range is off by up to
                 2^-25 of the largest weight, whatever its own size;
  6e-5 A         logits, exponentials and the sum (as in test_gpu_bounded.py);
  n 2^-24 A      adding n products in 32 bits."""
import torch

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def bound(out, mag, vsum, n, dtype):
    """out and mag of the 64-bit reference, vsum = sum_j |v_j| over the n visible positions."""
    u = U[dtype]
    tol = u * out.abs() + (2 * u * u + 6e-5 + n * 2.0 ** -24) * mag
    return tol + 2.0 ** -25 * (1 + vsum) if dtype == torch.float16 else tol
