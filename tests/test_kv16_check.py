"""CPU: errors that calls on the paged caches recorded, by the name of the cache."""
import pytest
import torch


@pytest.mark.parametrize("name", ["kv4", "kv16"])
@pytest.mark.parametrize("code,why", [(1, "timed out"), (6, "page table"), (7, "past the pool"), (99, "error 99")])
def test_recorded_errors(xtg, name, code, why):
    err = torch.tensor([code], dtype=torch.int32)
    check = getattr(xtg, f"{name}_check")
    with pytest.raises(xtg.XtgError, match=f"^{name}: .*{why}"):
        check(err)
    check(err)   # cleared
