"""Shared by the tests of the prompt attention and the 4-bit cache: inputs, and the bound their outputs are held to."""

import numpy as np
import torch

from oracle import serving

TYPES = {'fp16': torch.float16, 'bf16': torch.bfloat16}


def rounded(rng, shape, dtype, scale=1.0):
    """Normal values of a torch dtype on the CPU, and as float64."""
    t = torch.from_numpy(np.asarray(rng.standard_normal(shape) * scale, np.float32)).to(dtype)
    return t, t.double().numpy()


def check_attention(got, out, spread, size, vmax, keys, dtype):
    """got (float64) against the float64 result `out` within the bound that the kernel's roundings give, with
    u = eps / 2 of the type: the output rounded (u |out|); each weight rounded for the product with v, and their sum
    (2 u spread); scores summed in fp32 over at most 128 products and scaled (2 x 128 x 2^-24 size, twice: weight and
    sum), exponentials and fp32 sums of weights (2^-19 spread, keys x 2^-24 spread); fp16 weights below 2^-14 of at
    least 1 (keys x 2^-25 vmax) and outputs there (2^-25)."""
    u = torch.finfo(dtype).eps / 2
    with np.errstate(invalid='ignore'):
        tol = u * np.abs(out) + (2 * u + 2.0 ** -15 * size[..., None] + 2.0 ** -19 + keys * 2.0 ** -24) * spread \
            + keys * 2.0 ** -25 * vmax + 2.0 ** -25
        finite = np.isfinite(out)
        assert np.array_equal(np.isnan(got), np.isnan(out)) and np.array_equal(got[~finite & ~np.isnan(out)], out[~finite & ~np.isnan(out)])
        err = np.abs(got - out)[finite]
    assert (err <= tol[finite]).all(), f'max err {err.max():.3e}, worst ratio {(err / tol[finite]).max():.2f}'


def starts(lengths, dev):
    return torch.tensor([0, *np.cumsum(lengths)], dtype=torch.int64, device=dev)


def check_prompts(got, q, k, v, nq, nk, scale, causal, dtype):
    """Packed float64 inputs and the packed result of a prompt_attention call, sequence by sequence."""
    a = c = 0
    for x, y in zip(nq, nk):
        out, spread, size = serving.attend(q[a:a + x], k[c:c + y], v[c:c + y], scale, causal)
        vmax = np.abs(v[c:c + y][np.isfinite(v[c:c + y])]).max(initial=0)
        check_attention(got[a:a + x], out, spread, size, vmax, y, dtype)
        a, c = a + x, c + y


def to_device(cache, dev):
    from flash_whisper_amd.ext import KvQ4Cache

    return KvQ4Cache(*(torch.from_numpy(np.ascontiguousarray(c)).to(dev) for c in cache))


def same_bits(cache, want):
    """Every byte of a device cache against the oracle's."""
    return all(np.array_equal(t.cpu().numpy().view(np.uint8), np.ascontiguousarray(w).view(np.uint8))
               for t, w in zip(cache, want))
