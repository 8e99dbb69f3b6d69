"""Outputs of the batched serving calls that are their inputs, on a HIP runtime without a device."""
from test_serving_calls import INVALID, serving  # noqa: F401


def test_appended_queries_over_their_inputs(serving):  # noqa: F811
    names = "q+kin+vin+out+q_stride+num_rows+k_eq_v"
    cases = [  # 4 query heads of 64; the calls have room for 20 rows
        ("8192+4096+16384+8192+256+20+0", True),    # in place, row upon row
        ("8192+4096+16384+8192+512+20+0", False),   # rows of a packed matrix: a row's output lies on the next one's input
        ("8192+4096+16384+8192+512+1+0", True),     # one row
        ("8192+4096+16384+4096+256+20+0", False),   # on the keys
        ("8192+4096+16384+16384+256+20+0", False),  # on the values
        ("8192+4096+16384+16384+256+20+1", True),   # values that are not read
        ("8192+4096+16384+12288+512+20+0", True),
    ]
    for (values, fine), (st, _, why, kernels) in zip(cases, serving("append", *[(names, c[0]) for c in cases])):
        assert st == (0 if fine else INVALID) and bool(kernels) == fine, (values, st, why)
        assert fine or why.startswith("gh_kv8_append"), why


def test_nothing_to_append_over_its_inputs(serving):  # noqa: F811
    # no query heads: their arguments are not looked at; no rows: nothing is written
    assert serving("append", ("q+kin+out+num_q", "8192+4096+4096+0"))[0][0] == 0
    assert serving("append", ("q+out+num_rows", "8192+8192+0"))[0][0] == 0
