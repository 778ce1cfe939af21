"""Engine-side producers of the attention metadata."""

from voiceagent_amd.engine.metadata import (DecodeGraphMetadata, SequenceState, prepare_batch,
                                            prepare_batch_device, slot_of)

__all__ = ["DecodeGraphMetadata", "SequenceState", "prepare_batch",
           "prepare_batch_device", "slot_of"]
