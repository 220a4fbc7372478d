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


def test_the_polynomial_that_takes_a_share_of_the_exponentials():
    """2^x as the kernel's FMA steps compute it, with the coefficients of its source: 2.9e-6 and the rounding of four steps
    (4 * 2^-24) off at most, exactly 1 at 0, exactly 0 from -127 down."""
    import re

    import numpy as np
    from conftest import PKG_DIR
    body = (PKG_DIR / "csrc" / "attention_chunk.cuh").read_text().split("void ex2_poly2")[1].split("\n}")[0]
    coefficients = [np.float32(v) for v in re.findall(r"pack2\((0\.\d+|1\.0)f, \1f\)", body)]
    assert len(coefficients) == 5 and coefficients[-1] == 1
    f32, f64 = np.float32, np.float64

    def ex2(x):
        x = np.maximum(x.astype(f32), f32(-127))
        t = x + f32(12582912)
        f = x - (t - f32(12582912))
        p = np.full_like(x, coefficients[0])
        for c in coefficients[1:]:
            p = (p.astype(f64) * f + f64(c)).astype(f32)
        return (p.view(np.uint32) + (t.view(np.uint32) << np.uint32(23))).view(f32)

    x = np.concatenate([np.linspace(-126, 8, 2_000_001), np.arange(-126, 9)]).astype(f32)
    want = np.exp2(x.astype(f64))
    assert np.max(np.abs(ex2(x) - want) / want) < 2.9e-6 + 4 * 2.0 ** -24
    assert ex2(np.zeros(1, f32))[0] == 1
    assert (ex2(np.array([-127, -128, -1e30, -np.inf], f32)) == 0).all()


@pytest.mark.parametrize("scale", [2.0 ** 127, -(2.0 ** 127), 3.4e38, float("inf"), float("nan")])
def test_attention_chunk_refuses_scales_that_leave_f32(qasr, scale):
    """The softmax runs in powers of two, under scale * log2(e)."""
    with pytest.raises(qasr.DecoderError) as e:
        qasr.kernel_attention_chunk(0, 0, 0, A, 2048, A, 2048, 5, A, 9, A, 4, 8, 2, 16, 8, 1, A, A, A, 2, A, 1 << 40, scale=scale)
    assert e.value.status == 1 and "chunk attention" in str(e.value)
