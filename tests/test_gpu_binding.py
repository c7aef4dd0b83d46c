"""The compiled binding where a launch reports an error: it is raised, and the call is not made a second time."""

import ctypes

import pytest
import torch

from flash_whisper_amd import _lib

pytestmark = pytest.mark.gpu


@pytest.fixture
def ext(hip_device):
    """An ext of its own, whose calls through ctypes fail the test; the binding's entries are put back."""
    from flash_whisper_amd.ext import WhisperExt

    made = WhisperExt()
    assert made._bind is not None
    made._call = None
    yield made
    WhisperExt()


def _answer(ext, name, status, real):
    """The binding's entry `name` answers `status`, after the call itself (`real`) or without one; returns what counts the calls."""
    calls, entry = [], getattr(ext.lib, name)

    def stub(*args):
        calls.append(entry(*args) if real else 0)
        return status

    calls_it = ctypes.CFUNCTYPE(ctypes.c_int, *_lib.SIGNATURES[name][1])(stub)
    ext._kept = calls_it
    ext._bind.set_entry(name, ctypes.cast(calls_it, ctypes.c_void_p).value)
    return calls


def _calls(ext, dev):
    """A valid call of every op of the binding."""
    i64 = lambda *x: torch.tensor(x, dtype=torch.int64, device=dev)
    rows = lambda n, heads: torch.ones(n, heads, 64, dtype=torch.float16, device=dev)
    q, k, cu, pos = rows(3, 4), rows(3, 2), i64(0, 1, 3), i64(0, 0)
    q4, pages = ext.kv_q4_cache(2, 2, 64, 64), ext.kv_pages(4, 2, 16, 64)
    table = torch.zeros(3, 1, dtype=torch.int32, device=dev)
    x, ws = torch.ones(1, 8, device=dev), torch.empty(1 << 20, device=dev)
    return {'fw_prompt_attention': lambda: ext.prompt_attention(q, k, k, q.clone(), cu, cu, 0.125),
            'fw_kv_q4_append': lambda: ext.kv_q4_append(k, k, cu, pos, q4), 'fw_kv_q4_read': lambda: ext.kv_q4_read(q4, cu, pos, k, k.clone()),
            'fw_decode_attention_q4': lambda: ext.decode_attention_q4(q[:2], q4, i64(1, 2), q[:2].clone(), ws, 0.125),
            'fw_kv_page_map': lambda: ext.kv_page_map(i64(0, 0, 0), i64(0, 1, 2, 3), table, i64(0, 0, 0), table.view(-1).clone(), i64(3, 0), i64(0, 0, 0), 16),
            'fw_kv_page_append': lambda: ext.kv_page_append(k, k, i64(0, 1, 2), pages),
            'fw_decode_attention_paged': lambda: ext.decode_attention_paged(q, pages, table, i64(1, 1, 1), q.clone(), ws, 0.125),
            'fw_logits_rules': lambda: ext.logits_rules(x, x, tokens=i64(1), cu=i64(0, 1), repetition=x[0, :1])}


@pytest.mark.parametrize('name', ['fw_prompt_attention', 'fw_kv_q4_append', 'fw_kv_q4_read', 'fw_decode_attention_q4', 'fw_kv_page_map',
                                  'fw_kv_page_append', 'fw_decode_attention_paged', 'fw_logits_rules'])
def test_launch_error_is_raised(ext, hip_device, name):
    call = _calls(ext, hip_device)[name]
    call()
    calls = _answer(ext, name, _lib.FW_EHIP, real=False)
    with pytest.raises(_lib.FwError, match=f'{name}: .*status -2'):
        call()
    assert len(calls) == 1
    # an entry that refuses has launched nothing: the ctypes call reports it
    calls = _answer(ext, name, _lib.FW_EINVAL, real=False)
    with pytest.raises(TypeError):  # (which is taken away here)
        call()
    assert len(calls) == 1


def test_rules_in_place_once(ext, hip_device):
    """A launch that reports an error left before it has run all the same: logits that are their own output are ruled once."""
    i64 = lambda *x: torch.tensor(x, dtype=torch.int64, device=hip_device)
    x = torch.full((1, 8), 8.0, device=hip_device)
    calls = _answer(ext, 'fw_logits_rules', _lib.FW_EHIP, real=True)
    del ext._call  # (what a second call would go through)
    with pytest.raises(_lib.FwError):
        ext.logits_rules(x, x, tokens=i64(3), cu=i64(0, 1), repetition=torch.full((1,), 2.0, device=hip_device), bias_ids=i64(5),
                         bias=torch.ones(1, device=hip_device), cu_bias=i64(0, 1))
    assert calls == [_lib.FW_OK] and x[0].tolist() == [8, 8, 8, 4, 8, 9, 8, 8]

