"""The prefill's refusal of uneven head groups: its message names the rule (a per
cent sign in a format, read as a conversion, wrote through a stray pointer)."""
import ctypes

from mugen_amd import _capi


def test_uneven_head_groups_are_refused():
    a = _capi.GqaPrefillArgs()
    a.q = a.k = a.v = a.out = 0x1000
    a.n_tokens, a.n_heads, a.n_kv_heads, a.head_dim, a.kv_len = 4, 30, 4, 128, 4
    a.dtype = a.out_dtype = _capi.F16
    assert _capi.lib().mugen_attn_gqa_prefill(ctypes.byref(a), None) == _capi.E_INVALID
    assert _capi.lib().mugen_attn_last_error().decode() == "gqa_prefill: n_heads % n_kv_heads != 0"
