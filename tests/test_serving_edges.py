"""Refusals of the serving calls, without a GPU: scalar arguments are checked on the host before the device is touched."""
import pytest

A = 4096  # a stand-in for a device pointer, never read


@pytest.mark.parametrize("change", [
    dict(k_ptr=0), dict(v_ptr=0), dict(pool_ptr=0), dict(page_table_ptr=0), dict(row_slot_ptr=0), dict(row_pos_ptr=0),
    dict(row_count_ptr=0), dict(pool_pages=0), dict(max_slots=0), dict(max_pages=0), dict(max_pages=1 << 25), dict(layers=0),
    dict(layer=-1), dict(layer=2), dict(nkv=0), dict(nkv=(1 << 20) + 1), dict(rows_cap=0), dict(rows_cap=-1),
    dict(k_ptr=A + 8), dict(v_ptr=A + 2), dict(pool_ptr=A + 4),
])
def test_kv_append_planned_refuses_bad_arguments(qasr, change):
    a = dict(device=0, stream=0, k_ptr=A, v_ptr=A, pool_ptr=A, pool_pages=9, page_table_ptr=A, max_slots=4, max_pages=8,
             layers=2, nkv=8, layer=1, row_slot_ptr=A, row_pos_ptr=A, rows_cap=5, row_count_ptr=A)
    a.update(change)
    with pytest.raises(qasr.DecoderError) as e:
        qasr.kernel_kv_append_planned(**a)
    assert e.value.status == 1 and "planned kv append" in str(e.value)


def test_kv_append_planned_refuses_a_device_out_of_range(qasr):
    with pytest.raises(qasr.DecoderError) as e:
        qasr.kernel_kv_append_planned(99, 0, A, A, A, 9, A, 4, 8, 2, 8, 1, A, A, 5, A)
    assert e.value.status == 4
