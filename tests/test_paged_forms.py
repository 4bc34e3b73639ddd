"""Which kernel tree_attention takes, on the CPU (bml_diag_attn_tree_form): the
choice goes by what the caller says of its batch."""
import ctypes as C

import pytest


@pytest.fixture(scope="module")
def L():
    from bml_b200 import build
    build.build()
    import bml_b200._lib as lib
    return lib


FORMS = ["f32", "few", "warp", "umma", "umma32"]


def form(L, q, kv, n_tokens, group, d, n_seqs, n_live=0, max_new=0, positions=131072, n_kv=8):
    code = {"f32": L.BML_F32, "f16": L.BML_F16, "bf16": L.BML_BF16}
    f = C.c_int()
    st = L.lib().bml_diag_attn_tree_form(code[q], code[kv], n_tokens, group * n_kv, n_kv, d, 64, positions // 64, n_seqs, n_live,
                                         max_new, C.byref(f))
    assert st == L.BML_OK
    return FORMS[f.value]


@pytest.mark.parametrize("q,kv,many", [("bf16", "bf16", "umma"), ("f32", "f32", "umma32")])
def test_idle_and_narrow_requests_do_not_choose_the_kernel(L, q, kv, many):
    """A wide draft in a table of 64 places of which most are idle, or hold single
    tokens, takes the kernel that it takes alone."""
    assert form(L, q, kv, 64, 4, 128, 1) == many
    assert form(L, q, kv, 64, 4, 128, 64, n_live=1, max_new=64) == many
    assert form(L, q, kv, 60 + 4 * 64, 4, 128, 64, n_live=64, max_new=64) == many
    assert form(L, q, kv, 63 + 64, 4, 128, 64, n_live=64, max_new=64) == many


def test_32_bit_queries_over_16_bit_pages_go_by_the_average(L):
    assert form(L, "f32", "f16", 64, 4, 128, 1) == "warp"
    assert form(L, "f32", "f16", 64, 4, 128, 64, n_live=1, max_new=64) == "warp"
    assert form(L, "f32", "f16", 63 + 64, 4, 128, 64, n_live=64, max_new=64) == "few"


def test_narrow_batches_keep_their_kernel(L):
    """Single tokens, alone, among idle places, and beside a draft that is read a few times."""
    assert form(L, "bf16", "bf16", 64, 4, 128, 64) == "few"
    assert form(L, "bf16", "bf16", 3, 8, 64, 64, n_live=3, max_new=1) == "few"
    assert form(L, "bf16", "bf16", 63 + 8, 4, 128, 64, n_live=64, max_new=8) == "few"
    assert form(L, "f32", "f32", 64, 4, 128, 64, n_live=64, max_new=1) == "f32"
    # one short request in narrow tables: little work, whatever else the table holds
    assert form(L, "bf16", "bf16", 8, 8, 64, 1, positions=704, n_kv=4) == "warp"
    assert form(L, "bf16", "bf16", 8, 8, 64, 64, n_live=1, max_new=8, positions=704, n_kv=4) == "warp"
    # and without a hint the average over all requests
    assert form(L, "bf16", "bf16", 64, 4, 128, 64) == form(L, "bf16", "bf16", 64, 4, 128, 64, 64, 1)


def test_32_bit_pages_by_the_work(L):
    """Few rows, or little work for the longer start of the tcgen05 form, take row groups of 16."""
    one = dict(group=4, d=128, n_seqs=1)
    assert form(L, "f32", "f32", 5, positions=704, **one) == "f32"
    assert form(L, "f32", "f32", 30, positions=704, **one) == "umma32"
    assert form(L, "f32", "f32", 5, positions=2048, **one) == "f32"
    assert form(L, "f32", "f32", 16, positions=2048, **one) == "umma32"
    assert form(L, "f32", "f32", 5, positions=131072, **one) == "umma32"
    assert form(L, "f32", "f32", 4, positions=131072, **one) == "f32"
    assert form(L, "f32", "f32", 16, 8, 64, 1, positions=704, n_kv=4) == "f32"
    assert form(L, "f32", "f32", 16, 8, 64, 1, positions=4096, n_kv=4) == "umma32"
    # d = 64: two row groups of 16 at any size
    assert form(L, "f32", "f32", 64 * 4, 8, 64, 64, n_kv=4) == "f32"
    assert form(L, "f32", "f32", 64 * 5, 8, 64, 64, n_kv=4) == "umma32"
