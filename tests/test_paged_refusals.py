"""CPU checks of what the paged and sampling entry points refuse beyond the shapes (test_paged_rules.py): addresses and numbers that would go wrong on the device."""
import pytest

from test_paged_rules import A, BAD, L, calls, good  # noqa: F401


@pytest.mark.parametrize("what,field,which", [("batch", "dev_lengths", "awt"), ("batch", "dev_counts", "awt"), ("batch", "dev_pages", "awt"), ("batch", "dev_prefix_pages", "awt"),
                                              ("sampling", "dev_temperature", "s"), ("sampling", "dev_top_k", "s"), ("sampling", "dev_top_p", "s"), ("sampling", "dev_min_p", "s"),
                                              ("sampling", "dev_probs", "s"), ("sampling", "dev_tokens", "s")])
@pytest.mark.parametrize("off", [1, 2, 3])
def test_misaligned_arrays_are_refused(L, what, field, which, off):  # noqa: F811
    """Lengths, tables and settings between two words, in every call that reads them."""
    import torch
    d = good(L)
    setattr(d[what], field, A + off)
    got = dict(zip("awts", calls(L, d)))
    assert all(got[c] == BAD for c in which), got
    setattr(d[what], field, A + 4)  # a word's boundary is enough: what is refused then is that this is no device's memory
    got = dict(zip("awts", calls(L, d)))
    want = BAD if torch.cuda.is_available() else L.ERR_NO_DEVICE
    assert all(got[c] == want for c in which), got


@pytest.mark.parametrize("scale,fine", [(3e38, False), (-3e38, False), (2.4e38, False), (2.3e38, True), (-2.3e38, True), (1e-45, True)])
def test_scales_whose_exponents_overflow_are_refused(L, scale, fine):  # noqa: F811
    """exp(scale * x) is taken as a power of two: scale * log2(e) has to be a number."""
    import torch
    d = good(L)
    d["queries"].scale = scale
    got = calls(L, d)
    want = BAD if not fine or torch.cuda.is_available() else L.ERR_NO_DEVICE
    assert got[1] == got[2] == want
