"""What attention over an 8-bit cache may be off by on rows whose softmax has a
heavy key and a long tail, and the split of the softmax weights, on the CPU."""

import math

import torch

# A weight enters the products rounded to f16 (half a step, 2^-11 of itself), as a sum of
# three e5m2 parts: two cut off after three bits each, the third rounded at its third
# bit, so that at most half of the ninth bit is lost, 2^-9.
WEIGHT_STEP = 2.0 ** -9 + 2.0 ** -11
# The parts end at e5m2's smallest step, 2^-16, half of which is lost. A row's largest
# weight is at least 2^LEAST_TOP.
LEAST_TOP = 12
FLOOR = 2.0 ** (-17 - LEAST_TOP)


def split_weights(w):
    """The sum (f64) of the three e5m2 parts of weights w (f32, in [0, 57344))."""
    x = w.to(torch.float16)
    total = torch.zeros_like(w, dtype=torch.float64)
    for _ in range(2):
        part = (x.view(torch.int16) & -256).view(torch.float16)  # the upper byte of an f16 is an e5m2
        total += part.double()
        x = x - part
    part = ((x.view(torch.int16) + 128) & -256).view(torch.float16)
    return total + part.double()


def attend(q, k, v, v_codes, v_scales, seen):
    """(o, tolerance) of one head's rows, as `kv8_ref.attend` takes them. Every weight is
    off by a part of itself, and by FLOOR of the row's largest. The score's part: q enters
    as two e4m3 parts over a power of two that puts its largest element at 224 or above;
    half of the second part's smallest step, 2^-10, is lost, 2^-10 / 224 of that element;
    its f32 sums lose at most D steps of 2^-23; in log2 units and below 2^5 the factor's
    rounding, those of two sums and the exponential's stay below 2^-18. The f32 sums of weights and of the
    products: below 32 tiles' worth of steps a CTA and 74 parts to join at the lengths
    tested, 2^-13; the output 2^-8."""
    D = q.shape[1]
    s = (q @ k.T / math.sqrt(D)).masked_fill(~seen, -math.inf)
    p = torch.softmax(s, 1)
    p = torch.where(seen.any(1, keepdim=True), p, torch.zeros_like(p))
    o, mag = p @ v, p @ v.abs()
    # Each key's own score error, weighed as the key is; l's part is the mean of them.
    off = ((q.abs() @ k.abs().T) * D * 2.0 ** -23 + q.abs().amax(1, keepdim=True) * k.abs().sum(1) * (2.0 ** -10 / 224)) / math.sqrt(D)
    off = torch.where(seen, off + 2.0 ** -18, torch.zeros_like(off))
    mean = (p * off).sum(1, keepdim=True)
    scores = (p * off) @ v.abs() + mean * o.abs()
    floor = (p * v_scales).amax(1, keepdim=True) * FLOOR * (seen.double() @ v_codes.abs())
    return o, (mag * (WEIGHT_STEP + 2.0 ** -13) + scores + floor) * 1.01 + o.abs() * 2.0 ** -8
