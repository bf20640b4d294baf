// attention_stream_more.hip -- the kernel of attention_stream.hip for launches with first tokens beside a window and with prefixes
// that sequences share; in a file of its own so that both compile side by side.
#define IQ4XS_ATTENTION_MORE
#include "attention_stream.hip"
