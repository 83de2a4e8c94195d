"""Inputs on which an attention's weights of 11 bits show and weights of 22 bits do not.  Only tests use this.

Heavy keys come in pairs whose scores differ by one step of a 256th of a power of two and whose values are each other's negatives: a
context is some 2^-11 of the sum of weight times |value|, so neither its own rounding nor the sums' hides what the weights are off
by.  Between the heavy keys lie light ones, 2^-200 of the heavy ones and less, which fp32 holds as zeros: they add nothing, and no
error."""
import torch

HEADS, D = 8, 64
ALPHA = 2.0 ** -8 / 1.4426950408889634


def sequence(g, keys, heavy):
    """q [HEADS, D], k and v [keys, D] int8 of one token, the first and last heavy / 2 keys heavy."""
    q, k, v = torch.zeros(HEADS, D), torch.zeros(keys, D), torch.zeros(keys, D)
    q[:, 0], q[:, 1] = torch.arange(9, 9 + HEADS), 1
    q[:, 2:6] = 127
    k[:, 2:6] = -128
    at = torch.cat([torch.arange(heavy // 2), torch.arange(keys - heavy // 2, keys)])
    k[at, 2:6] = 0
    k[at, 0] = torch.randint(-30, 31, (heavy // 2,), generator=g).repeat_interleave(2).float()
    k[at[0::2], 1] = torch.randint(-8, 8, (heavy // 2,), generator=g).float()
    k[at[1::2], 1] = k[at[0::2], 1] + 1
    v[at[0::2]] = torch.randint(0, 2, (heavy // 2, D), generator=g).float() * 200 - 100
    v[at[1::2]] = -v[at[0::2]]
    return q.to(torch.int8), k.to(torch.int8), v.to(torch.int8), at


def wanted(q, k, v, at):
    """As ``_paged_oracle.attention`` of one token, of the heavy keys alone."""
    s = float(torch.tensor(ALPHA, dtype=torch.float32)) * (q.double() @ k[at].double().T)
    w = torch.softmax(s, 1)
    return w @ v[at].double(), w @ v[at].double().abs(), s.abs().amax(1, keepdim=True) * 1.4427
