"""What a model in precision 'mx4' says about itself (host logic: no handle is built)."""
import warnings

import pytest
import torch

from uit_mobile_amd.models.uit import UitkSetupWarning
from test_gpu_mx4_engine import build


def warning_of(precision, monkeypatch):
    m = build(precision=precision)
    monkeypatch.setattr(type(m), "_build_handle", lambda self, idx: object())
    with warnings.catch_warnings(record=True) as seen:
        warnings.simplefilter("always")
        m._handle_obj(torch.device("cuda", 0))
        m.refresh()
        m._handle_obj(torch.device("cuda", 0))
    seen = [w for w in seen if issubclass(w.category, UitkSetupWarning)]
    assert len(seen) == 1                                                    # once per model
    return str(seen[0].message)


def test_the_warning_of_the_general_engine_names_what_the_precision_does(monkeypatch):
    mx4, f32 = warning_of("mx4", monkeypatch), warning_of("f32", monkeypatch)
    assert "GENERAL fp32 engine" in f32 and "4 bits" not in f32
    assert "fp32 engine" not in mx4 and "order of operations" not in mx4
    assert "4 bits" in mx4 and "outside the parity budget" in mx4 and "logits" in mx4


@pytest.mark.parametrize("precision", ["mx4", "f32"])
def test_what_belongs_to_the_other_kernels_is_refused_with_the_right_reason(precision):
    m = build(precision=precision)
    for call in (m.calibrate, m.self_check, lambda: m.set_option("split_pe", 1)):
        with pytest.raises(NotImplementedError, match="this model runs on the general") as e:
            call()
        assert ("4 bits" in str(e.value)) == (precision == "mx4") and ("rounds nothing" in str(e.value)) == (precision == "f32")
