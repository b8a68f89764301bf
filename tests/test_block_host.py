"""Host-side parts of the operators around the experts that need no GPU: the descriptions' layout, workspace
sizes, and null arguments (each refused before anything touches a device)."""

import pytest

import vastloom_b200 as vb


def test_packed_descriptions_have_the_structures_layout():
    n = list(range(1, 16))
    assert bytes(vb._AddRmsNormDesc(*n[:12], 31, 32, 2, 1, 0.5, 0)) == vb._ADD_RMS_NORM_PACK(*n[:12], 31, 32, 2, 1, 0.5, 0)
    assert (bytes(vb._AddRmsNormGradDesc(*n[:14], 31, 32, 2, 1, 0.5, 0)) ==
            vb._ADD_RMS_NORM_GRAD_PACK(*n[:14], 31, 32, 2, 1, 0.5, 0))
    assert bytes(vb._SortTokensDesc(*n, 31, 32, 33, 34, 2, 0)) == vb._SORT_TOKENS_PACK(*n, 31, 32, 33, 34, 2, 0)
    assert bytes(vb._CombineDesc(*n[:8], 31, 32, 33, 34, 2, 1)) == vb._COMBINE_PACK(*n[:8], 31, 32, 33, 34, 2, 1)
    assert bytes(vb._CombineGradDesc(*n[:9], 31, 32, 33, 34, 2, 1)) == vb._COMBINE_GRAD_PACK(*n[:9], 31, 32, 33, 34, 2, 1)
    assert bytes(vb._Int8Epilogue(*n[:3], 5, 0.5)) == vb._INT8_EPILOGUE_PACK(*n[:3], 5, 0.5)


SIZES = [0, 1, 2, 7, 31, 64, 100, 147, 148, 149, 295, 296, 300, 443, 444, 445, 1000, 1411, 4095, 4096, 4097, 65536, 1 << 20]


def test_norm_workspace_never_falls():
    for a in SIZES[1:]:
        by_rows = [vb.add_rms_norm_grad_workspace_bytes(r, a) for r in SIZES]
        by_cols = [vb.add_rms_norm_grad_workspace_bytes(a, c) for c in SIZES[1:]]
        assert by_rows == sorted(by_rows) and by_cols == sorted(by_cols)


def test_sort_workspace_never_falls():
    for k in (1, 2, 8, 64):
        for E in (1, 8, 256, 1024):
            sizes = [vb.sort_tokens_workspace_bytes(T, k, E) for T in SIZES + [1 << 24]]
            assert sizes == sorted(sizes)
            for T in SIZES:
                assert vb.sort_tokens_workspace_bytes(T, k, E) <= vb.sort_tokens_workspace_bytes(T, k + 1, E + 1)
            assert vb.sort_tokens_workspace_bytes(1 << 20, k, E) < 1 << 30


@pytest.mark.parametrize("name", ["vlb_add_rms_norm_device", "vlb_add_rms_norm_grad_device", "vlb_sort_tokens_device",
                                  "vlb_combine_device", "vlb_combine_grad_device"])
def test_null_handles_are_errors(name):
    assert getattr(vb.load_library(), name)(None, None, None) == 1


def test_int8_epilogue_of_a_null_handle_is_an_error():
    lib = vb.load_library()
    assert lib.vlb_int8_linear_act_device(None, None, None, None) == 1
    assert lib.vlb_int8_linear_act_device(None, None, vb._INT8_EPILOGUE_PACK(0, 0, 0, 0, 0.0), None) == 1
