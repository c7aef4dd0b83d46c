"""Every way in which the prompt attention shares out its rows, named by the library for the sizes at hand: against the
float64 oracle, within the bound of serving_tools.check_attention."""

import numpy as np
import pytest
import torch

from flash_whisper_amd import _lib
from serving_tools import TYPES, check_prompts, rounded, starts

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def ext(hip_device):
    from flash_whisper_amd.ext import load_ext

    return load_ext()


# form: the queries and keys of the sequences, heads and key/value heads. Partial blocks and tiles in each; single waves with
# sequences of many tiles among the short ones; blocks of 128 rows over more than 1500 keys and over few
FORMS = {'waves': (_lib.PROMPT_WAVES, [150] + [1] * 20, [200] + [3] * 20, 8, 4), 'waves_last': (_lib.PROMPT_WAVES, [1, 0, 2] * 9 + [333], [1, 5, 0] * 9 + [333], 6, 2),
         'long_wide': (_lib.PROMPT_128_ROWS, [1300, 1201], [1500, 2100], 40, 20), 'short_wide': (_lib.PROMPT_128_ROWS, [60, 1, 133] * 22, [100, 1, 140] * 22, 40, 20),
         'two_parts': (_lib.PROMPT_2_PARTS, [300, 70], [900, 601], 20, 20), 'two_short_parts': (_lib.PROMPT_2_SHORT_PARTS, [150, 33, 90], [150, 70, 210], 20, 20),
         'eight_parts': (_lib.PROMPT_8_PARTS, [4, 37, 1], [1000, 531, 777], 8, 2)}


def _form(ext, nq, nk, heads, kv_heads, dim, causal):
    return ext.lib.fw_prompt_attention_form(len(nq), sum(nq), sum(nk), heads, kv_heads, dim, causal)


def _check_some(ext, dev, form, dim, kind, causal, edit=None):
    """The call of a form; the query heads of the first and the last key/value head are compared."""
    want, nq, nk, heads, kv_heads = FORMS[form]
    assert _form(ext, nq, nk, heads, kv_heads, dim, causal) == want
    dtype, rng, group = TYPES[kind], np.random.default_rng(dim + causal), heads // kv_heads
    q, q64 = rounded(rng, (sum(nq), heads, dim), dtype)
    k, k64 = rounded(rng, (sum(nk), kv_heads, dim), dtype)
    v, v64 = rounded(rng, (sum(nk), kv_heads, dim), dtype)
    if edit:
        edit(k, v, nk)
        k64, v64 = k.double().numpy(), v.double().numpy()
    out = torch.full((sum(nq), heads, dim), float('nan'), dtype=dtype, device=dev)
    ext.prompt_attention(q.to(dev), k.to(dev), v.to(dev), out, starts(nq, dev), starts(nk, dev), dim ** -0.5, causal)
    got = out.double().cpu().numpy()
    assert edit or not np.isnan(got).any()
    for h in (0, kv_heads - 1):
        own = slice(h * group, (h + 1) * group)
        check_prompts(got[:, own], q64[:, own], k64[:, h:h + 1], v64[:, h:h + 1], nq, nk, dim ** -0.5, causal, dtype)


@pytest.mark.parametrize('kind, dim', [('fp16', 64), ('bf16', 64), ('fp16', 128), ('bf16', 128)])
@pytest.mark.parametrize('causal', [True, False])
@pytest.mark.parametrize('form', FORMS)
def test_prompt_forms(ext, hip_device, form, causal, kind, dim):
    _check_some(ext, hip_device, form, dim, kind, causal)


@pytest.mark.parametrize('kind, dim', [('fp16', 64), ('bf16', 128)])
@pytest.mark.parametrize('causal', [True, False])
@pytest.mark.parametrize('form', FORMS)
def test_prompt_forms_no_numbers(ext, hip_device, form, causal, kind, dim):
    """Infinities and NaN near the end of each sequence, whose last causal queries alone see them, and in its middle."""
    def edit(k, v, nk):
        for end, n in zip(np.cumsum(nk), nk):
            if n > 20:
                k[end - 2, 0, 9] = float('inf')
                v[end - 1, -1, 3], v[end - 3, -1, 4], v[end - 2, -1, dim - 1] = float('nan'), float('inf'), float('-inf')
                v[end - 17, -1, 5], v[end - n // 2, -1, 7] = float('inf'), float('nan')

    _check_some(ext, hip_device, form, dim, kind, causal, edit)
