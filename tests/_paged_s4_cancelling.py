"""Inputs for the 4-bit cache on which an attention's weights of 11 bits show and weights of 22 bits do not.  Only tests use this.

As for the int8 cache (``_paged_cancelling``): heavy keys come in pairs whose scores differ by one step of a 256th of a power of two and
whose values are each other's negatives, so a context is some 2^-11 of the sum of weight times |value|; the light keys between
them, 2^-100 of the heavy ones and less, add nothing.  Codes are around z = 7; steps are powers of two, one for all keys and one
for all values, so scores are whole multiples of the step of the keys and fp32 holds them as they are."""
import torch

Z, K_STEP, V_STEP = 7, 2.0, 16.0
ALPHA = 2.0 ** -8 / K_STEP / 1.4426950408889634
LIGHT = 36          # columns that tell light keys from heavy ones: 36 * 127 * 7 is more than 100 * 256


def sequence(g, keys, heavy, new, q_heads, d):
    """q int8 [new, q_heads, d], codes less z of k and v [keys, d] of a sequence's last ``new`` tokens, and which keys are heavy: half
    of them the first ones, half the last that all the tokens see."""
    q, k, v = torch.zeros(new, q_heads, d), torch.zeros(keys, d), torch.zeros(keys, d)
    q[..., :3] = torch.randint(5, 17, (new, q_heads, 3), generator=g).float()
    q[..., 3] = 1
    q[..., d - LIGHT + 4:] = q[..., 4:8] = 127
    k[:, d - LIGHT + 4:] = k[:, 4:8] = -Z
    seen = keys - new + 1
    at = torch.cat([torch.arange(heavy // 2), torch.arange(seen - heavy // 2, seen)])
    k[at] = 0
    k[at, :3] = torch.randint(-7, 9, (heavy // 2, 3), generator=g).float().repeat_interleave(2, 0)
    k[at[0::2], 3] = torch.randint(-7, 8, (heavy // 2,), generator=g).float()
    k[at[1::2], 3] = k[at[0::2], 3] + 1
    v[at[0::2]] = torch.randint(0, 2, (heavy // 2, d), generator=g).float() * 14 - 7
    v[at[1::2]] = -v[at[0::2]]
    return q.to(torch.int8), k, v, at


def codes(x):
    """Bytes [..., d / 2] of codes less z [..., d]."""
    u = (x + Z).to(torch.uint8)
    half = u.shape[-1] // 2
    return u[..., :half] + 16 * u[..., half:]


def word(step):
    return int(torch.tensor(step, dtype=torch.float16).view(torch.int16)) | Z


def wanted(q, k, v, at):
    """(context, sum of weight times |value|, largest |score| in powers of two) as ``_paged_oracle.attention`` has them, of the heavy
    keys alone; q [..., d]."""
    s = float(torch.tensor(ALPHA, dtype=torch.float32)) * K_STEP * (q.double() @ k[at].double().T)
    w = torch.softmax(s, -1)
    value = V_STEP * v[at].double()
    return w @ value, w @ value.abs(), s.abs().amax(-1, keepdim=True) * 1.4427
