"""Arguments of the cache, attention and verification calls that are refused before any launch (no GPU)."""
import pytest

import viper_amd as va

torch = pytest.importorskip("torch")


def test_verify_draft_refuses_host_tensors():
    """Tensors that are all on the host agree on their device, and their addresses mean nothing on the GPU."""
    z = lambda *s, dt=torch.int32: torch.zeros(s, dtype=dt)
    with pytest.raises(ValueError, match="GPU"):
        va.verify_draft(z(2, 3, 100, dt=torch.bfloat16), z(2, 2), z(2, 3, dt=torch.float32), z(2, 3), z(2),
                        workspace=z(va.verify_workspace_bytes(2, 3, 100), dt=torch.uint8))
