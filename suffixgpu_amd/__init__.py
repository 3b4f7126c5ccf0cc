"""MI355X (gfx950) SuffixGPU drafter.

Drop-in for zip95297/SuffixGPU's draft path (suffix_gpu/__init__.py:1-4):
``SuffixGPUDrafter`` with propose / update_state / propose_with_update /
harvest_finished / poll, running hand-written HIP kernels from
``libsuffixgpu_amd.so`` (built by ``python -m suffixgpu_amd.build``).  Beside
it, for the target model that checks the drafts: ``KV4Cache``, a paged cache
held in 4 bits with its attention, and ``verify_draft``.
"""

from suffixgpu_amd.kv4 import KV4Cache
from suffixgpu_amd.proposer import SuffixGPUDrafter
from suffixgpu_amd.verify import verify_draft

__version__ = "0.1.2"
__all__ = ["SuffixGPUDrafter", "KV4Cache", "verify_draft", "__version__"]
