"""paged_decode_attention_fp8's scale: what would not be finite in the kernel's units (times
log2 e) is refused before a launch; the scores would be NaN."""

from evo2_flash_amd import _lib


def test_scales_past_the_kernels_units_are_refused():
    lib, n, at = _lib.lib(), None, 4096  # (an aligned address that is never read)

    def attend(scale):  # (B 0 returns before the launch, behind the check of the scale)
        return lib.evo2_paged_decode_attention_fp8(at, 1024, 1024, 128, at, 4096, 2048, at, 4096, 2048, at, 2, 1, at, 2, 1, 8,
                                                   at, 4, 4, 0, at, at, 1 << 30, at, 1024, 1024, 128, 0, 1, 8, 2, 128, scale, n)

    for scale in (1e-40, 0.125, 1.0, 2.3e38):
        assert attend(scale) == 0
    for scale in (2.4e38, 3.4e38, float("inf"), float("nan"), 0.0, -1.0):
        assert attend(scale) == 1 and b"scale" in lib.evo2_last_error()
