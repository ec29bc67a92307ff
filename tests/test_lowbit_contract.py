"""The decode operators in fewer bits, what can be told without a GPU: what the binding keeps alive, which
forms the GPU tests reach."""
import ctypes as C
import gc
import weakref

import pytest

import g2hip
import test_lowbit_addresses as addresses
import test_lowbit_contract_gpu as gpu
import test_lowbit_gpu as base


class Buf(g2hip.DevBuf):
    """A buffer that owns no memory."""

    def __init__(self, ptr):
        self.ptr, self.nbytes = ptr, 0

    def free(self):
        self.ptr = None


@pytest.mark.parametrize("name", ["ctx", "ctx_len", "bias_id", "bias", "mask"])
def test_rules_keep_their_buffers(name):
    """A structure of rules holds addresses: buffers that only it refers to live as long as it does."""
    buf = Buf(0x1000)
    alive = weakref.ref(buf)
    rules = g2hip.logit_rules(**{name: buf}, max_ctx=3, n_bias=2)
    del buf
    gc.collect()
    assert alive() is not None and getattr(rules, name) == alive().ptr == 0x1000
    del rules
    gc.collect()
    assert alive() is None


def test_every_form_of_a_product_meets_outliers():
    forms = addresses.q4_form
    assert {forms(M, N, K)[0] for M, N, K, _ in gpu.OUTLIERS} == {forms(M, N, K)[0] for M, N, K, _ in base.product_cases()}
    assert len({(forms(M, N, K)[0], G) for M, N, K, G in gpu.OUTLIERS}) == 33


def test_every_form_of_the_rules_is_tested():
    fn = g2hip._lib.g2i_logits_form
    fn.argtypes = [C.c_int, C.c_int, C.POINTER(C.c_int)]
    seen = set()
    cases = [m for m in base.test_rules.pytestmark if m.name == "parametrize"][0].args[1]
    for R, V in cases + gpu.WIDE:
        parts = C.c_int()
        wide = fn(R, V, C.byref(parts))
        assert (parts.value - 1) * (8192 if wide else 1024) < V <= parts.value * (8192 if wide else 1024)
        assert not (R, V) in gpu.WIDE or wide
        seen.add((bool(wide), parts.value > 1))
    assert len(seen) == 4
