"""The serving calls' refusals and sizes without a GPU: every scalar argument is checked on the host before the
device is touched, so each wrong call comes back as a status with a message (the pointers given are
never read)."""
import pytest

A = 4096  # a stand-in for a device pointer, well aligned


def _plan(**kw):
    a = dict(device=0, stream=0, seq_slot_ptr=A, kv_len_ptr=A, new_len_ptr=A, n_seqs=2, max_slots=4, page_table_ptr=A,
             max_pages=8, free_pages_ptr=A, pool_pages=32, free_count_ptr=A, kv_len_out_ptr=A, free_count_out_ptr=A,
             cu_rows_ptr=A, row_slot_ptr=A, row_pos_ptr=A, rows_cap=16, status_ptr=A)
    a.update(kw)
    return a


@pytest.mark.parametrize("change", [
    dict(seq_slot_ptr=0), dict(kv_len_ptr=0), dict(page_table_ptr=0), dict(free_pages_ptr=0), dict(free_count_ptr=0),
    dict(kv_len_out_ptr=0), dict(free_count_out_ptr=0), dict(cu_rows_ptr=0), dict(row_slot_ptr=0), dict(row_pos_ptr=0),
    dict(status_ptr=0), dict(n_seqs=0), dict(n_seqs=-1), dict(n_seqs=8193), dict(max_slots=0), dict(max_slots=65537),
    dict(max_pages=0), dict(max_pages=1 << 25), dict(pool_pages=-1), dict(rows_cap=-1),
])
def test_kv_plan_refuses_bad_arguments(qasr, change):
    with pytest.raises(qasr.DecoderError) as e:
        qasr.kernel_kv_plan(**_plan(**change))
    assert e.value.status == 1 and "kv plan" in str(e.value)


@pytest.mark.parametrize("change", [
    dict(seq_slot_ptr=0), dict(kv_len_ptr=0), dict(page_table_ptr=0), dict(free_pages_ptr=0), dict(free_count_ptr=0),
    dict(kv_len_out_ptr=0), dict(free_count_out_ptr=0), dict(status_ptr=0), dict(n_seqs=0), dict(n_seqs=8193),
    dict(max_slots=0), dict(max_pages=0), dict(pool_pages=-1),
])
def test_kv_release_refuses_bad_arguments(qasr, change):
    a = {k: v for k, v in _plan().items()
         if k not in ("new_len_ptr", "cu_rows_ptr", "row_slot_ptr", "row_pos_ptr", "rows_cap")}
    a.update(change)
    with pytest.raises(qasr.DecoderError) as e:
        qasr.kernel_kv_release(**a)
    assert e.value.status == 1 and "kv release" in str(e.value)


@pytest.mark.parametrize("change", [
    dict(q_ptr=0), dict(out_ptr=0), dict(pool_ptr=0), dict(page_table_ptr=0), dict(seq_slot_ptr=0), dict(cu_rows_ptr=0),
    dict(kv_len_ptr=0), dict(ws_ptr=0), dict(rows=0), dict(rows=-3), dict(n_seqs=0), dict(pool_pages=0), dict(max_slots=0),
    dict(max_pages=0), dict(max_pages=1 << 25), dict(layers=0), dict(layer=-1), dict(layer=2), dict(nkv=0), dict(nq=0),
    dict(nq=12), dict(nq=8 * 17), dict(q_ld=2047), dict(out_ld=2040), dict(q_ld=2052), dict(out_ld=2050),
    dict(q_ptr=A + 2), dict(out_ptr=A + 8), dict(pool_ptr=A + 4), dict(ws_ptr=A + 128), dict(type=2), dict(type=-1),
    dict(scale=float("nan")), dict(scale=float("inf")),
    dict(pool_pages=2**20, layers=2),  # 2^20 x 2 x 2 x 8 x 64 = 2^31 rows: past the row coordinates
])
def test_attention_chunk_refuses_bad_arguments(qasr, change):
    a = dict(device=0, stream=0, type=0, q_ptr=A, q_ld=2048, out_ptr=A, out_ld=2048, rows=5, pool_ptr=A, pool_pages=9,
             page_table_ptr=A, max_slots=4, max_pages=8, layers=2, nq=16, nkv=8, layer=1, seq_slot_ptr=A, cu_rows_ptr=A,
             kv_len_ptr=A, n_seqs=2, ws_ptr=A, ws_bytes=1 << 40)
    a.update(change)
    with pytest.raises(qasr.DecoderError) as e:
        qasr.kernel_attention_chunk(**a)
    assert e.value.status == 1 and "chunk attention" in str(e.value)


def test_attention_chunk_check_refuses_bad_workspaces(qasr):
    for ptr in (0, A + 8):
        with pytest.raises(qasr.DecoderError) as e:
            qasr.kernel_attention_chunk_check(0, 0, ptr)
        assert e.value.status == 1


def test_devices_out_of_range_are_refused(qasr):
    with pytest.raises(qasr.DecoderError):
        qasr.kernel_attention_chunk_workspace(-1)
    with pytest.raises(qasr.DecoderError):
        qasr.kernel_attention_chunk_workspace(99)
    with pytest.raises(qasr.DecoderError) as e:
        qasr.kernel_kv_plan(**_plan(device=99))
    assert e.value.status == 4


def test_w4_packed_bytes(qasr):
    # codes in 2 KB units of 32 rows x 128 columns, 2 bytes of scale and 1 of zero point per row and group
    assert qasr.kernel_w4_packed_bytes(32, 128, 128) == 2048 + 64
    assert qasr.kernel_w4_packed_bytes(33, 128, 128) == 2 * (2048 + 64)
    assert qasr.kernel_w4_packed_bytes(32, 128, 32, True) == 2048 + 4 * 32 * 3
    assert qasr.kernel_w4_packed_bytes(1, 96, 32) == 2048 + 4 * 64  # columns 96..127 are padding
    for n_out, k, g in [(0, 64, 64), (-1, 64, 64), (16, 0, 64), (16, 64, 16), (16, 96, 64), (16, 64, 128), (16, 64, 0)]:
        with pytest.raises(qasr.DecoderError):
            qasr.kernel_w4_packed_bytes(n_out, k, g)


@pytest.mark.parametrize("change", [dict(codes_ptr=0), dict(scale_ptr=0), dict(packed_ptr=0), dict(packed_ptr=A + 8),
                                    dict(group=48), dict(k=130), dict(n_out=0)])
def test_pack_w4_refuses_bad_arguments(qasr, change):
    a = dict(device=0, stream=0, codes_ptr=A, scale_ptr=A, zero_ptr=None, n_out=16, k=128, group=64, packed_ptr=A)
    a.update(change)
    with pytest.raises(qasr.DecoderError) as e:
        qasr.kernel_pack_w4(**a)
    assert e.value.status == 1 and "w4 pack" in str(e.value)


@pytest.mark.parametrize("change", [
    dict(packed_ptr=0), dict(x_ptr=0), dict(out_ptr=0), dict(rows=0), dict(rows=65), dict(ldx=120), dict(ldx=130),
    dict(ldo=15), dict(packed_ptr=A + 8), dict(x_ptr=A + 2), dict(out_ptr=A + 1), dict(type=3), dict(group=16),
])
def test_gemv_w4_refuses_bad_arguments(qasr, change):
    a = dict(device=0, stream=0, type=0, packed_ptr=A, has_zero=False, n_out=16, k=128, group=64, x_ptr=A, ldx=128, rows=1,
             out_ptr=A, ldo=16)
    a.update(change)
    with pytest.raises(qasr.DecoderError) as e:
        qasr.kernel_gemv_w4(**a)
    assert e.value.status == 1 and "w4 gemv" in str(e.value)
