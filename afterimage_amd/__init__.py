"""afterimage_amd: MI355X-native lossless BF16 weight decoder for Afterimage's
compressed-store format. See afterimage_amd.runtime for the decode API, and
its attention and kv_cache modules for what runs between the decoded projections."""
__version__ = "0.1.0"
