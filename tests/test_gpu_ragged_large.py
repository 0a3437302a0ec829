"""The packed prefill over keys and values that do not fit L2 together, where its blocks
go kv head by kv head: each sequence's rows are those of a prefill of it alone."""
import pytest

from test_gpu_ragged import Z16, _packed, _run, _same_as_alone

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hq,hkv,nq,nk", [
    (24, 8, [9000, 700, 0, 5001, 2600], None),       # groups of 3
    (8, 8, [300, 1, 4000], [9000, 6001, 4000]),      # a head for each, chunks behind prefixes
    (32, 2, [600, 130], [40000, 30001]),             # groups of 16
])
@pytest.mark.parametrize("window", [None, Z16])
def test_ragged_rows_past_l2_are_those_of_the_sequence_alone(hq, hkv, nq, nk, window):
    import atflash
    q, k, v, cq, ck = _packed(nq, nk or nq, hq, hkv, hq)
    assert ck[-1] * hkv * 512 > 64 << 20
    got = _run(q, k, v, cq, ck, window_table=window)
    _same_as_alone(got, q, k, v, cq, ck, causal=True, window_table=window)
    assert atflash.check_device_errors() == 0
