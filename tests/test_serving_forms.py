"""Which attention kernel the plan takes for the cases that run on the GPU (kv8_forms.py), on a
HIP runtime without a device."""
import pytest

from kv8_forms import PROMPTS, STREAMS
from test_serving_calls import serving  # noqa: F401

NAMES = ("num_q", "num_kv", "head_dim", "page_tokens", "num_seqs", "num_rows", "max_rows", "window", "max_pages", "max_kv", "num_pages")


def launched(serving, values):  # noqa: F811
    (st, need, why, kernels), = serving("attn", ("+".join(NAMES), "+".join(str(v) for v in values)))
    assert st == 0, why
    return kernels[0][0], need


@pytest.mark.parametrize("nq,H,D,page,rows,past,window,max_pages,kernel", STREAMS)
def test_plans_of_codes_by_the_caches(serving, nq, H, D, page, rows, past, window, max_pages, kernel):  # noqa: F811
    assert launched(serving, (nq, H, D, page, len(rows), sum(rows), max(rows), window, max_pages, 0, 1000))[0] == kernel


@pytest.mark.parametrize("nq,H,D,page,rows,past,window,bounds,kernel", PROMPTS)
def test_plans_of_prompts(serving, nq, H, D, page, rows, past, window, bounds, kernel):  # noqa: F811
    per = max(-(-(p + r) // page) for p, r in zip(past, rows))
    name, need = launched(serving, (nq, H, D, page, len(rows), *bounds, window, per, 0, 1000))
    assert name == kernel and need == 0


def test_every_kernel_of_the_attention_is_run():
    forms = {case[-1] for case in STREAMS + PROMPTS}
    for nl in (1, 2, 4, 8):
        for r in ("", "r"):
            assert "gh_kv8_attn_l%d%ss_k" % (nl, r) in forms and "gh_kv8_rows_l%d%s_k" % (nl, r) in forms
