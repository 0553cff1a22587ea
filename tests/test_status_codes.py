"""What a code in the kernels' status word is reported as (no GPU: the word is a tensor on the host)."""
import pytest
import torch

from gogguf_b200.csrc import tcgen05_gemm as tc
from gogguf_b200.csrc.build import KernelError


@pytest.mark.parametrize("code, said", [(29, "attn_prefill_tc refused"), (69, "mixed_head_attention refused"), (70, "attn_decode_shared refused"), (54, "attn_decode_shared met"),
                                        (71, "bounded wait"), (79, "bounded wait"), (12, "bounded wait")])
def test_codes_name_what_happened(monkeypatch, code, said):
    word = torch.tensor([code], dtype=torch.int32)
    monkeypatch.setitem(tc._status, torch.device("cpu"), word)
    with pytest.raises(KernelError, match=said):
        tc.check_status("cpu")
    assert int(word) == 0                    # reported once
    tc.check_status("cpu")


def test_a_kernel_over_shared_prefixes_has_a_code_of_its_own():
    """No other kernel writes 70."""
    import os
    import re
    folder = os.path.join(os.path.dirname(tc.__file__))
    writers = [f for f in sorted(os.listdir(folder)) if f.endswith((".cu", ".cuh"))
               and re.search(r"atomicCAS\(status, 0, 70\)", open(os.path.join(folder, f)).read())]
    assert writers == ["attention_shared.cu"]
