"""The scale bytes of the 4-bit cache: 252 is the largest that every code of bf16's range can have."""
import numpy as np

from oracle import kv4_oracle as KO
from oracle import mxfp4_oracle as O


def test_the_largest_scale():
    codes = np.tile(np.arange(16, dtype=np.uint8), 2)[None]
    for scale in range(256):
        values = KO.dequantize(codes, np.array([[scale]], np.uint8))
        if scale > 252:
            assert np.isnan(values).all()
        else:
            assert np.array_equal(O.bf16_to_f32(O.f32_to_bf16(values.astype(np.float32))), values)
    assert 6 * 2.0 ** (252 - 127) < 2.0 ** 128 <= 4 * 2.0 ** (253 - 127)
    top = np.full((1, 32), 0x7F7F, np.uint16)           # the largest finite bf16
    assert KO.quantize(O.bf16_to_f32(top))[1].tolist() == [[252]]
