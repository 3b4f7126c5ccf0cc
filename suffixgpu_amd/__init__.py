"""MI355X (gfx950) SuffixGPU drafter.

Drop-in for zip95297/SuffixGPU's draft path (suffix_gpu/__init__.py:1-4):
``SuffixGPUDrafter`` with propose / update_state / propose_with_update /
harvest_finished / poll, running hand-written HIP kernels from
``libsuffixgpu_amd.so`` (built by ``python -m suffixgpu_amd.build``).  Beside
it, for the target model that checks the drafts: ``KV4Cache``, a paged cache
held in 4 bits with its attention, ``PagePool``, its page tables, ``verify_draft``
and ``token_logprobs``.
"""

from suffixgpu_amd.kv4 import KV4Cache
from suffixgpu_amd.logprobs import token_logprobs
from suffixgpu_amd.pages import PagePool
from suffixgpu_amd.proposer import SuffixGPUDrafter
from suffixgpu_amd.verify import verify_draft

__version__ = "0.1.2"
__all__ = ["SuffixGPUDrafter", "KV4Cache", "PagePool", "verify_draft",
           "token_logprobs", "__version__"]
